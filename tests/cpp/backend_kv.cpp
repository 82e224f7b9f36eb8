// Test of the C++ Backend adapter's rotary positions and 8-bit paged cache (include/halo_mi355x_backend.hpp,
// MiBackend::rope and kv8_*): two sequences take their pages, are rotated, written, read back and attended to, one is
// forked and the pool compacted, each step against plain loops in 64 bits; then the error mapping.
//
// Built by __graft_entry__.build(); run by tests/test_backend_kv_cpp.py (GPU) with no arguments, or with --list (no GPU
// needed).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <memory>
#include <set>
#include <span>
#include <string>
#include <utility>
#include <vector>

#include "../../include/halo_mi355x.h"
#include "../../include/halo_mi355x_backend.hpp"

namespace hb = halo_mi::backend;

namespace {

int g_failures = 0;
int g_checks = 0;

void check(bool ok, const std::string& what) {
    ++g_checks;
    if (!ok) {
        ++g_failures;
        std::printf("FAIL %s\n", what.c_str());
    }
}

int code_of(const std::function<void()>& f) {
    try {
        f();
    } catch (const hb::Error& e) {
        return static_cast<int>(e.code());
    }
    return -1;
}

struct Device {
    hb::MiBackend& be;
    hb::Stream& st;
    template <class T>
    std::unique_ptr<hb::Buffer> up(const std::vector<T>& v) {
        auto b = be.allocate(v.size() * sizeof(T), hb::Tier::Vram);
        be.upload(st, hb::TensorRef::of(*b), std::as_bytes(std::span<const T>(v)));
        st.wait();
        return b;
    }
    template <class T>
    std::vector<T> down(const hb::Buffer& b) {
        std::vector<T> v(b.bytes() / sizeof(T));
        be.download(st, hb::TensorRef::of(b), std::as_writable_bytes(std::span<T>(v)));
        st.wait();
        return v;
    }
};

std::vector<float> normal(uint64_t seed, size_t n) {
    std::vector<float> v(n);
    halo_mi_fill_normal(seed, v.data(), n, 0.0f, 1.0f);
    return v;
}

constexpr uint32_t kLayers = 2, kLayer = 1, kHeads = 4, kKvHeads = 2, kDim = 64, kBlock = 16, kPages = 12, kSlots = 4, kWidth = 4;

hb::TensorRef of(const std::unique_ptr<hb::Buffer>& b) { return hb::TensorRef::of(*b); }

void serving(hb::MiBackend& be, hb::Stream& st) {
    Device dev{be, st};
    const std::vector<int32_t> lens{21, 5};
    const uint32_t rows = 26;
    auto pool = be.allocate(kPages * halo_mi_kv_page_bytes(kLayers, kKvHeads, kDim, kBlock), hb::Tier::Vram);
    auto refs = dev.up(std::vector<int32_t>(kPages, 0)), slot_lens = dev.up(std::vector<int32_t>(kSlots, 0));
    auto tables = dev.up(std::vector<int32_t>(kSlots * kWidth, -1));
    const hb::Kv8Cache cache{of(pool), kPages, kLayers, kKvHeads, kDim, kBlock};
    const hb::Kv8State state{of(refs), of(slot_lens), of(tables), kSlots, kWidth};

    // pages
    auto slots = dev.up(std::vector<int32_t>{0, 1}), new_lens = dev.up(lens);
    be.kv8_resize(st, {cache, state, of(slots), of(new_lens), 2});
    st.wait();
    const auto table = dev.down<int32_t>(*tables);
    check(std::set<int32_t>{table[0], table[1], table[kWidth]} == std::set<int32_t>({0, 1, 2}), "kv8_resize gives the lowest pages");
    check(dev.down<int32_t>(*slot_lens) == std::vector<int32_t>({21, 5, 0, 0}), "kv8_resize sets the lengths");

    // rotary positions of q and k, in place
    const uint32_t rot = 32;
    std::vector<double> freqs(rot / 2);
    float factor = 0.0f;
    check(halo_mi_rope_freqs(rot, 10000.0, nullptr, freqs.data(), &factor) == HALO_MI_OK, "rope_freqs");
    std::vector<int32_t> positions;
    for (int32_t n : lens)
        for (int32_t i = 0; i < n; ++i) positions.push_back(i);
    const auto q0 = normal(1, rows * kHeads * kDim), k0 = normal(2, rows * kKvHeads * kDim), v0 = normal(3, rows * kKvHeads * kDim);
    auto q = dev.up(q0), k = dev.up(k0), v = dev.up(v0), pos = dev.up(positions), fr = dev.up(freqs);
    hb::RopeTableArgs ra;
    ra.parts[0] = {of(q), of(q), kHeads};
    ra.parts[1] = {of(k), of(k), kKvHeads};
    ra.n_parts = 2, ra.n_tokens = rows, ra.head_dim = kDim, ra.rot_dims = rot, ra.positions = of(pos), ra.freqs = of(fr), ra.factor = factor;
    be.rope(st, ra);
    st.wait();
    const auto q1 = dev.down<float>(*q), k1 = dev.down<float>(*k);
    double worst = 0.0;
    const auto rotated = [&](const std::vector<float>& in, const std::vector<float>& out, uint32_t heads) {
        for (uint32_t t = 0; t < rows; ++t)
            for (uint32_t h = 0; h < heads; ++h) {
                const float *x = &in[(t * heads + h) * kDim], *y = &out[(t * heads + h) * kDim];
                for (uint32_t i = 0; i < rot / 2; ++i) {
                    const double a = positions[t] * freqs[i], c = std::cos(a), s = std::sin(a);
                    const double size = std::hypot(x[i], x[i + rot / 2]);
                    // two fp32 factors of the angle and three roundings: under 8 half steps
                    worst = std::max(worst, std::abs(y[i] - (x[i] * c - x[i + rot / 2] * s)) / (size * std::ldexp(8.0, -24)));
                    worst = std::max(worst, std::abs(y[i + rot / 2] - (x[i + rot / 2] * c + x[i] * s)) / (size * std::ldexp(8.0, -24)));
                }
                for (uint32_t i = rot; i < kDim; ++i) check(x[i] == y[i], "rope copies the elements behind rot_dims");
            }
    };
    rotated(q0, q1, kHeads);
    rotated(k0, k1, kKvHeads);
    check(worst <= 1.0, "rope is the rotation: " + std::to_string(worst));

    // write, read, attention; layer 1, tables as the pages' owner left them
    auto starts = dev.up(std::vector<int32_t>{0, 21, 26});
    const hb::Kv8Batch batch{of(tables), of(slot_lens), of(starts), 2, rows, kWidth};
    hb::Kv8WriteArgs wa;
    wa.cache = cache, wa.layer = kLayer, wa.batch = batch, wa.k = of(k), wa.v = of(v);
    be.kv8_write(st, wa);
    auto k_back = be.allocate(k1.size() * 4, hb::Tier::Vram), v_back = be.allocate(v0.size() * 4, hb::Tier::Vram);
    hb::Kv8ReadArgs rd;
    rd.cache = cache, rd.layer = kLayer, rd.batch = batch, rd.k = of(k_back), rd.v = of(v_back);
    be.kv8_read(st, rd);
    auto out = be.allocate(q1.size() * 4, hb::Tier::Vram), ws = be.allocate(1u << 20, hb::Tier::Vram);
    hb::Kv8AttentionArgs aa;
    aa.cache = cache, aa.layer = kLayer, aa.batch = batch, aa.q = of(q), aa.out = of(out), aa.n_heads = kHeads, aa.workspace = of(ws);
    be.kv8_attention(st, aa);
    st.wait();
    const auto kr = dev.down<float>(*k_back), vr = dev.down<float>(*v_back), o = dev.down<float>(*out);
    const uint32_t first[] = {0, 21};
    double step = 0.0;
    for (int x = 0; x < 2; ++x) {
        const auto& in = x ? v0 : k1;
        const auto& got = x ? vr : kr;
        for (uint32_t s = 0; s < 2; ++s)
            for (uint32_t h = 0; h < kKvHeads; ++h)
                for (uint32_t b = 0; b < (uint32_t)lens[s]; b += kBlock) {
                    double amax = 0.0;
                    const uint32_t e = std::min<uint32_t>(b + kBlock, lens[s]);
                    for (int pass = 0; pass < 2; ++pass)
                        for (uint32_t t = b; t < e; ++t)
                            for (uint32_t d = 0; d < kDim; ++d) {
                                const size_t i = ((first[s] + t) * kKvHeads + h) * kDim + d;
                                if (pass == 0) amax = std::max<double>(amax, std::abs(in[i]));
                                // half a step of amax / 127, and the roundings of scale, quotient and product
                                else step = std::max(step, std::abs((double)in[i] - got[i]) / (amax / 127 * 0.5 + amax * std::ldexp(4.0, -24)));
                            }
                }
    }
    check(step <= 1.0, "kv8_write and kv8_read keep values to half a step: " + std::to_string(step));
    double off = 0.0;
    for (uint32_t s = 0; s < 2; ++s)
        for (uint32_t t = 0; t < (uint32_t)lens[s]; ++t)
            for (uint32_t h = 0; h < kHeads; ++h) {
                const float* qr = &q1[((first[s] + t) * kHeads + h) * kDim];
                std::vector<double> p(t + 1);
                double top = -1e300, sum = 0.0, size = 0.0;
                for (uint32_t j = 0; j <= t; ++j) {
                    const float* kj = &kr[((first[s] + j) * kKvHeads + h / 2) * kDim];
                    double dot = 0.0, abs = 0.0;
                    for (uint32_t d = 0; d < kDim; ++d) dot += (double)qr[d] * kj[d], abs += std::abs((double)qr[d] * kj[d]);
                    p[j] = dot / 8, size = std::max(size, abs / 8), top = std::max(top, p[j]);
                }
                for (double& x : p) sum += x = std::exp(x - top);
                // a score is off by q's 2^-22 and the sum of kDim products; a weight by that, twice (it and the sum), its
                // own 2^-22 and 4 roundings of the exponent's argument, up to 2^5, in 24 bits; sums of t + 1 terms
                const double bound = 2 * size * (std::ldexp(1.0, -22) + kDim * std::ldexp(1.0, -24)) + 2 * std::ldexp(1.0, -22) +
                                     2 * 4 * 32 * std::ldexp(1.0, -24) + 2 * (t + 2) * std::ldexp(1.0, -24);
                for (uint32_t d = 0; d < kDim; ++d) {
                    double y = 0.0, abs = 0.0;
                    for (uint32_t j = 0; j <= t; ++j) {
                        const double vj = vr[((first[s] + j) * kKvHeads + h / 2) * kDim + d];
                        y += p[j] / sum * vj, abs += p[j] / sum * std::abs(vj);
                    }
                    off = std::max(off, std::abs(o[((first[s] + t) * kHeads + h) * kDim + d] - y) / (abs * bound + 1e-30));
                }
            }
    check(off <= 1.0, "kv8_attention is the softmax over the cached tokens: " + std::to_string(off));

    // fork, grow the copy, free the source, compact
    auto src = dev.up(std::vector<int32_t>{0}), dst = dev.up(std::vector<int32_t>{2});
    be.kv8_fork(st, {cache, state, of(src), of(dst), 1});
    auto grown = dev.up(std::vector<int32_t>{33});
    be.kv8_resize(st, {cache, state, of(dst), of(grown), 1});
    st.wait();
    auto now = dev.down<int32_t>(*tables);
    check(now[2 * kWidth] == now[0] && now[2 * kWidth + 1] != now[1] && now[2 * kWidth + 2] >= 0, "kv8_fork shares whole pages only");
    check(dev.down<int32_t>(*refs)[now[0]] == 2, "kv8_fork counts the holders");
    auto zero = dev.up(std::vector<int32_t>{0});
    be.kv8_resize(st, {cache, state, of(src), of(zero), 1});
    auto live = dev.up(std::vector<uint32_t>{99});
    be.kv8_compact(st, {cache, state, of(live)});
    st.wait();
    check(dev.down<uint32_t>(*live)[0] == 4, "kv8_compact counts the live pages");
    now = dev.down<int32_t>(*tables);
    check(std::set<int32_t>{now[kWidth], now[2 * kWidth], now[2 * kWidth + 1], now[2 * kWidth + 2]} == std::set<int32_t>({0, 1, 2, 3}),
          "kv8_compact moves them to the front");
    // the second sequence, wherever its page is now, reads as before
    auto starts1 = dev.up(std::vector<int32_t>{0, 0, 5});
    rd.batch.row_starts = of(starts1), rd.batch.n_rows = 5;
    be.kv8_read(st, rd);
    st.wait();
    const auto again = dev.down<float>(*k_back);
    check(std::equal(again.begin(), again.begin() + 5 * kKvHeads * kDim, kr.begin() + 21 * kKvHeads * kDim), "the moved page keeps its bytes");
    // a page copied whole
    auto one = dev.up(std::vector<int32_t>{now[kWidth]}), free_page = dev.up(std::vector<int32_t>{9});
    be.kv8_copy_pages(st, {cache, {}, of(one), of(free_page), 1});
    st.wait();
    const auto bytes = dev.down<uint8_t>(*pool);
    const size_t page = halo_mi_kv_page_bytes(kLayers, kKvHeads, kDim, kBlock);
    check(std::memcmp(&bytes[9 * page], &bytes[now[kWidth] * page], page) == 0, "kv8_copy_pages copies whole pages");

    // ---- errors ----
    const auto refused = [&](hb::ErrorCode want, const char* what, const std::function<void()>& f) {
        check(code_of(f) == (int)want, std::string(what) + " is refused");
    };
    const auto bad = [&](auto args, auto change) {
        change(args);
        return args;
    };
    refused(hb::ErrorCode::Unsupported, "a quantized q", [&] { be.kv8_attention(st, bad(aa, [](auto& x) { x.type = hb::DType::Q8_0; })); });
    refused(hb::ErrorCode::Unsupported, "a head_dim of 80", [&] { be.kv8_attention(st, bad(aa, [](auto& x) { x.cache.head_dim = 80; })); });
    refused(hb::ErrorCode::Config, "an unknown variant", [&] { be.kv8_attention(st, bad(aa, [](auto& x) { x.kernel.variant_id = 31; })); });
    refused(hb::ErrorCode::Kernel, "a pool too small", [&] { be.kv8_attention(st, bad(aa, [](auto& x) { x.cache.n_pages = kPages + 1; })); });
    refused(hb::ErrorCode::Kernel, "out over q", [&] { be.kv8_attention(st, bad(aa, [&](auto& x) { x.out = of(q); })); });
    refused(hb::ErrorCode::Kernel, "heads not a multiple", [&] { be.kv8_attention(st, bad(aa, [](auto& x) { x.n_heads = 3; })); });
    refused(hb::ErrorCode::Kernel, "too few lengths", [&] { be.kv8_write(st, bad(wa, [](auto& x) { x.batch.n_seqs = 5; })); });
    refused(hb::ErrorCode::Kernel, "layer 2 of 2", [&] { be.kv8_write(st, bad(wa, [](auto& x) { x.layer = 2; })); });
    refused(hb::ErrorCode::Kernel, "an odd rot_dims", [&] { be.rope(st, bad(ra, [](auto& x) { x.rot_dims = 31; })); });
    refused(hb::ErrorCode::Unsupported, "three parts", [&] { be.rope(st, bad(ra, [](auto& x) { x.n_parts = 3; })); });
    const std::vector<std::byte> image(pool->bytes());
    auto frozen = be.import_host_readonly(image);
    refused(hb::ErrorCode::Kernel, "a read-only pool", [&] { be.kv8_write(st, bad(wa, [&](auto& x) { x.cache.pool = of(frozen); })); });
    auto other = hb::make_mi355x_backend(0);
    auto foreign = other->allocate(pool->bytes(), hb::Tier::Vram);
    refused(hb::ErrorCode::Kernel, "another backend's pool", [&] { be.kv8_read(st, bad(rd, [&](auto& x) { x.cache.pool = of(foreign); })); });

    // what the device finds is reported by wait(), or left in the caller's word
    auto wrong = dev.up(std::vector<int32_t>(kSlots * kWidth, 77));
    rd.batch.tables = of(wrong);
    be.kv8_read(st, rd);
    refused(hb::ErrorCode::Kernel, "a page out of range", [&] { st.wait(); });
    check(code_of([&] { st.wait(); }) == -1, "the status is reported once");
    auto word = dev.up(std::vector<uint32_t>{0xFFu});
    rd.status = of(word);
    be.kv8_read(st, rd);
    check(code_of([&] { st.wait(); }) == -1 && dev.down<uint32_t>(*word)[0] == hb::kStatusBadIndex, "a status word of the caller's");
    auto many = dev.up(std::vector<int32_t>{64, 64}), both = dev.up(std::vector<int32_t>{0, 3});
    be.kv8_resize(st, {cache, state, of(both), of(many), 2});
    st.wait();
    auto two = dev.up(std::vector<int32_t>{1});
    be.kv8_resize(st, {cache, state, of(two), of(many), 1});
    refused(hb::ErrorCode::Memory, "a sequence that finds no page", [&] { st.wait(); });
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--list") == 0) {
        std::printf("backend_kv\n");
        return 0;
    }
    try {
        auto be = hb::make_mi355x_backend(0);
        auto st = be->create_stream();
        const std::pair<hb::OpId, uint32_t> ids[] = {{hb::OpId::Rope, 51}, {hb::OpId::Kv8Write, 52}, {hb::OpId::Kv8Read, 53},
                                                     {hb::OpId::Kv8Attention, 54}, {hb::OpId::Kv8Pages, 55}};
        for (const auto& [op, id] : ids) check(be->variants(op).size() == 1 && be->variants(op)[0].id == id, "the variants' ids are pinned");
        serving(*be, *st);
    } catch (const std::exception& e) {
        std::printf("FAIL exception: %s\n", e.what());
        ++g_failures;
    }
    std::printf("backend_kv: %d checks, %d failures\n", g_checks, g_failures);
    return g_failures ? 1 : 0;
}
