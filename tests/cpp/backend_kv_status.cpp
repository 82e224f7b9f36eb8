// What ops of one stream find wrong on the device between two wait()s, of several kinds at once: every kind is thrown, one a
// wait() (include/halo_mi355x_backend.hpp, the paged cache's ops and GET_ROWS).
//
// Built by __graft_entry__.build(); run by tests/test_backend_kv_status_cpp.py (GPU) with no arguments, or with --list (no
// GPU needed).
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <memory>
#include <span>
#include <string>
#include <vector>

#include "../../include/halo_mi355x.h"
#include "../../include/halo_mi355x_backend.hpp"

namespace hb = halo_mi::backend;

namespace {

int g_failures = 0;

void check(bool ok, const std::string& what) {
    if (ok) return;
    ++g_failures;
    std::printf("FAIL %s\n", what.c_str());
}

// The code that f throws (-1: none); `text` receives what it says.
int code_of(const std::function<void()>& f, std::string* text = nullptr) {
    try {
        f();
    } catch (const hb::Error& e) {
        if (text) *text = e.what();
        return static_cast<int>(e.code());
    }
    return -1;
}

hb::TensorRef of(const std::unique_ptr<hb::Buffer>& b) { return hb::TensorRef::of(*b); }

template <class T>
std::unique_ptr<hb::Buffer> up(hb::MiBackend& be, hb::Stream& st, const std::vector<T>& v) {
    auto b = be.allocate(v.size() * sizeof(T), hb::Tier::Vram);
    be.upload(st, of(b), std::as_bytes(std::span<const T>(v)));
    st.wait();
    return b;
}

void several_kinds(hb::MiBackend& be, hb::Stream& st) {
    constexpr uint32_t kPages = 2, kSlots = 2, kWidth = 4, kDim = 64, kCols = 256, kRows = 4;
    auto pool = be.allocate(kPages * halo_mi_kv_page_bytes(1, 1, kDim, 16), hb::Tier::Vram);
    auto refs = up(be, st, std::vector<int32_t>(kPages, 0)), lens = up(be, st, std::vector<int32_t>(kSlots, 0));
    auto tables = up(be, st, std::vector<int32_t>(kSlots * kWidth, -1));
    const hb::Kv8Cache cache{of(pool), kPages, 1, 1, kDim, 16};
    const hb::Kv8State state{of(refs), of(lens), of(tables), kSlots, kWidth};
    auto stray = up(be, st, std::vector<int32_t>{9}), zero = up(be, st, std::vector<int32_t>{0}), much = up(be, st, std::vector<int32_t>{60});
    auto row = be.allocate(kCols * 4, hb::Tier::Vram);
    const uint64_t rb = halo_mi_row_bytes(static_cast<uint32_t>(hb::DType::Q8_0), kCols);
    auto table = up(be, st, std::vector<uint8_t>(kRows * rb, 0));

    hb::GetRowsArgs gr;
    gr.type = hb::DType::Q8_0, gr.table = of(table), gr.ids = of(stray), gr.out = of(row), gr.n_rows = kRows, gr.cols = kCols, gr.n_ids = 1;
    const auto bad_row = [&] { be.get_rows(st, gr); };
    const auto bad_slot = [&] { be.kv8_resize(st, {cache, state, of(stray), of(much), 1}); };
    const auto no_page = [&] { be.kv8_resize(st, {cache, state, of(zero), of(much), 1}); };
    const int kernel = (int)hb::ErrorCode::Kernel, memory = (int)hb::ErrorCode::Memory;
    std::string text;

    bad_slot(), no_page();
    check(code_of([&] { st.wait(); }, &text) == kernel && text.find("paged cache") != std::string::npos, "a slot out of range is thrown: " + text);
    check(code_of([&] { st.wait(); }) == memory, "pages that ran out in the same interval are thrown by the next wait()");
    check(code_of([&] { st.wait(); }) == -1, "each once");

    no_page(), bad_row(), bad_slot();
    check(code_of([&] { st.wait(); }, &text) == kernel && text.find("GET_ROWS") != std::string::npos, "GET_ROWS's id is thrown: " + text);
    no_page();  // again, before the rest was thrown
    check(code_of([&] { st.wait(); }, &text) == kernel && text.find("paged cache") != std::string::npos, "the slot is thrown: " + text);
    check(code_of([&] { st.wait(); }) == memory, "the pages are thrown");
    check(code_of([&] { st.wait(); }) == -1, "the stream is clean then");

    // a stream's bits are its own
    auto other = be.create_stream();
    bad_slot(), no_page();
    check(code_of([&] { other->wait(); }) == -1, "another stream's wait() does not throw for them");
    check(code_of([&] { st.wait(); }) == kernel && code_of([&] { st.wait(); }) == memory && code_of([&] { st.wait(); }) == -1, "its own does");
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--list") == 0) {
        std::printf("backend_kv_status\n");
        return 0;
    }
    try {
        auto be = hb::make_mi355x_backend(0);
        auto st = be->create_stream();
        several_kinds(*be, *st);
    } catch (const std::exception& e) {
        std::printf("FAIL exception: %s\n", e.what());
        ++g_failures;
    }
    std::printf("backend_kv_status: %d failures\n", g_failures);
    return g_failures ? 1 : 0;
}
