// Test of the C++ Backend adapter's head norms, 8-bit products and linear attention (include/halo_mi355x_backend.hpp,
// MiBackend::norm_rope, quantize_rows, gemm_i8, linear_attention): a projection held in 8 bits makes rows whose heads are normed and
// rotated and then attended to, each step against plain loops in 64 bits; then the error mapping.
//
// Built by __graft_entry__.build(); run by tests/test_backend_layer_cpp.py (GPU) with no arguments, or with --list (no GPU
// needed).
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <memory>
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

hb::TensorRef of(const std::unique_ptr<hb::Buffer>& b) { return hb::TensorRef::of(*b); }

// part of a buffer of rows: from `offset` elements on, rows `stride` elements apart
hb::TensorRef part(const std::unique_ptr<hb::Buffer>& b, uint64_t offset, uint64_t stride) {
    hb::TensorRef t = of(b);
    t.offset = offset * 4, t.bytes = b->bytes() - offset * 4, t.row_stride = stride * 4;
    return t;
}

constexpr uint32_t kRows = 26, kIn = 200, kHeads = 4, kKHeads = 2, kDim = 64, kSlots = 3;
constexpr uint32_t kOut = (kHeads + 2 * kKHeads) * kDim;  // q and k of kKHeads heads, v of kHeads

void layer(hb::MiBackend& be, hb::Stream& st) {
    Device dev{be, st};
    // ---- 8-bit rows and their product, into rows of q, k and v side by side
    const auto xh = normal(1, kRows * kIn), wh = normal(2, kOut * kIn);
    const uint32_t pad = (kIn + 15) / 16 * 16;
    auto x = dev.up(xh), w = dev.up(wh);
    auto xc = be.allocate(kRows * pad, hb::Tier::Vram), wc = be.allocate(kOut * pad, hb::Tier::Vram);
    auto xs = be.allocate(kRows * 4, hb::Tier::Vram), ws = be.allocate(kOut * 4, hb::Tier::Vram);
    auto y = be.allocate(kRows * kOut * 4, hb::Tier::Vram);
    const hb::QuantizeRowsArgs qx{hb::DType::F32, of(x), of(xc), of(xs), kRows, kIn};
    be.quantize_rows(st, qx);
    be.quantize_rows(st, {hb::DType::F32, of(w), of(wc), of(ws), kOut, kIn});
    const hb::GemmI8Args ga{hb::DType::F32, of(wc), of(ws), of(xc), of(xs), of(y), kOut, kIn, kRows};
    be.gemm_i8(st, ga);
    const auto xq = dev.down<int8_t>(*xc), wq = dev.down<int8_t>(*wc);
    const auto xf = dev.down<float>(*xs), wf = dev.down<float>(*ws), yh = dev.down<float>(*y);
    bool codes = true, products = true;
    for (uint32_t t = 0; t < kRows; ++t) {
        float most = 0.0f;
        for (uint32_t i = 0; i < kIn; ++i) most = std::max(most, std::fabs(xh[t * kIn + i]));
        codes = codes && xf[t] == most / 127.0f;
        for (uint32_t i = 0; i < pad; ++i) codes = codes && xq[t * pad + i] == (i < kIn ? (int)std::nearbyint((double)xh[t * kIn + i] / (double)xf[t]) : 0);
        for (uint32_t n = 0; n < kOut; ++n) {
            int32_t sum = 0;
            for (uint32_t i = 0; i < kIn; ++i) sum += (int)xq[t * pad + i] * (int)wq[n * pad + i];
            products = products && yh[t * kOut + n] == xf[t] * wf[n] * (float)sum;
        }
    }
    check(codes, "quantize_rows gives the nearest codes of the largest value's scale");
    check(products, "gemm_i8 is the exact sum with both scales");

    // ---- norms and positions of q and k where they lie
    std::vector<double> freqs(kDim / 2);
    float factor = 0.0f;
    check(halo_mi_rope_freqs(kDim, 10000.0, nullptr, freqs.data(), &factor) == HALO_MI_OK, "rope_freqs");
    std::vector<int32_t> positions;
    for (int32_t i = 0; i < (int32_t)kRows; ++i) positions.push_back(i < 21 ? i : 100 + i);
    const auto weights = normal(3, kDim);
    auto pos = dev.up(positions), fr = dev.up(freqs), nw = dev.up(weights);
    hb::NormRopeArgs na;
    na.rope = {hb::DType::F32, false, {}, 2, kRows, kDim, kDim, of(pos), of(fr), factor};
    na.rope.parts[0] = {part(y, 0, kOut), part(y, 0, kOut), kKHeads};
    na.rope.parts[1] = {part(y, kKHeads * kDim, kOut), part(y, kKHeads * kDim, kOut), kKHeads};
    na.norm_w[0] = of(nw);
    na.norm_w[1] = of(nw);
    be.norm_rope(st, na);
    const auto zh = dev.down<float>(*y);
    double worst = 0.0;
    bool kept = true;
    for (uint32_t t = 0; t < kRows; ++t)
        for (uint32_t h = 0; h < kHeads + 2 * kKHeads; ++h) {
            const float *a = &yh[t * kOut + h * kDim], *b = &zh[t * kOut + h * kDim];
            if (h >= 2 * kKHeads) {
                kept = kept && std::memcmp(a, b, kDim * 4) == 0;
                continue;
            }
            double sum = 0.0;
            for (uint32_t i = 0; i < kDim; ++i) sum += (double)a[i] * a[i];
            const double inv = 1.0 / std::sqrt(sum / kDim + na.eps);
            for (uint32_t i = 0; i < kDim / 2; ++i) {
                const double angle = positions[t] * freqs[i], c = std::cos(angle), s = std::sin(angle);
                const double u = a[i] * inv * weights[i], v = a[i + kDim / 2] * inv * weights[i + kDim / 2];
                // the sum's kDim roundings reach the root halved, and a dozen more follow; rotated, two such numbers add up
                const double tol = (kDim / 2 + 12) * std::ldexp(1.0, -24) * (std::fabs(u) + std::fabs(v));
                worst = std::max({worst, std::fabs(b[i] - (u * c - v * s)) / tol, std::fabs(b[i + kDim / 2] - (v * c + u * s)) / tol});
            }
        }
    check(worst <= 1.0, "norm_rope is the norm and the rotation: " + std::to_string(worst));
    check(kept, "norm_rope leaves v alone");

    // ---- linear attention: a prompt that begins here, in slot 2, and 5 more tokens of the sequence in slot 0
    const auto sh = normal(4, (size_t)kSlots * kHeads * kDim * kDim);
    std::vector<float> decays(kRows * kHeads);
    for (size_t i = 0; i < decays.size(); ++i) decays[i] = -0.01f * (float)(i % 13);
    auto state = dev.up(sh), after = dev.up(sh), decay = dev.up(decays), out = be.allocate(kRows * kHeads * kDim * 4, hb::Tier::Vram);
    auto slots = dev.up(std::vector<int32_t>{2, 0}), starts = dev.up(std::vector<int32_t>{0, 21, 26}), lens = dev.up(std::vector<int32_t>{21, 40});
    hb::LinearAttentionArgs la;
    la.n_heads = kHeads, la.n_k_heads = kKHeads, la.k_dim = la.v_dim = kDim, la.n_slots = kSlots;
    la.state = of(state), la.state_out = of(after), la.slots = of(slots), la.row_starts = of(starts), la.seq_lens = of(lens);
    la.n_seqs = 2, la.n_rows = kRows, la.max_rows = 21;
    la.q = part(y, 0, kOut), la.k = part(y, kKHeads * kDim, kOut), la.v = part(y, 2 * kKHeads * kDim, kOut), la.out = of(out), la.decay = of(decay);
    be.linear_attention(st, la);
    st.wait();
    const auto oh = dev.down<float>(*out), ah = dev.down<float>(*after);
    check(dev.down<float>(*state) == sh, "linear_attention keeps the states before the call");
    double worst_out = 0.0, worst_state = 0.0;
    for (uint32_t s = 0; s < 2; ++s) {
        const uint32_t slot = s ? 0 : 2, r0 = s ? 21 : 0, r1 = s ? 26 : 21;
        for (uint32_t h = 0; h < kHeads; ++h) {
            const size_t at = ((size_t)slot * kHeads + h) * kDim * kDim;
            // S and, beside it, the sum of what its terms are at most: errors are counted against that
            std::vector<double> S(kDim * kDim, 0.0), M(kDim * kDim, 0.0);
            if (s)
                for (uint32_t i = 0; i < kDim * kDim; ++i) S[i] = sh[at + i], M[i] = std::fabs(sh[at + i]);
            for (uint32_t t = r0; t < r1; ++t) {
                const float *q = &zh[t * kOut + h / 2 * kDim], *k = q + kKHeads * kDim, *v = &zh[t * kOut + (2 * kKHeads + h) * kDim];
                const double fade = std::exp((double)decays[t * kHeads + h]);
                for (uint32_t i = 0; i < kDim; ++i)
                    for (uint32_t j = 0; j < kDim; ++j) {
                        S[i * kDim + j] = fade * S[i * kDim + j] + (double)k[i] * v[j];
                        M[i * kDim + j] = fade * M[i * kDim + j] + std::fabs((double)k[i] * v[j]);
                    }
                for (uint32_t j = 0; j < kDim; ++j) {
                    double o = 0.0, m = 0.0;
                    for (uint32_t i = 0; i < kDim; ++i) o += S[i * kDim + j] * q[i], m += M[i * kDim + j] * std::fabs(q[i]);
                    // 32 tokens' sums of 64 terms in pieces of 2^-24, at most 128 roundings of 2^-24 on any term
                    worst_out = std::max(worst_out, std::fabs(oh[(t * kHeads + h) * kDim + j] - o / 8.0) / (128 * std::ldexp(1.0, -24) * m / 8.0));
                }
            }
            for (uint32_t i = 0; i < kDim * kDim; ++i)
                worst_state = std::max(worst_state, std::fabs(ah[at + i] - S[i]) / (64 * std::ldexp(1.0, -24) * M[i] + 1e-30));
        }
    }
    check(worst_out <= 1.0, "linear_attention's out: " + std::to_string(worst_out));
    check(worst_state <= 1.0, "linear_attention's states: " + std::to_string(worst_state));
    const size_t slot = (size_t)kHeads * kDim * kDim;
    check(std::memcmp(&ah[slot], &sh[slot], slot * 4) == 0, "a slot of no sequence keeps its bytes");
    // in place
    la.state_out = {};
    be.linear_attention(st, la);
    check(dev.down<float>(*state) == ah && dev.down<float>(*out) == oh, "linear_attention in place is bitwise the same");

    // ---- errors ----
    const auto refused = [&](hb::ErrorCode want, const char* what, const std::function<void()>& f) {
        check(code_of(f) == (int)want, std::string(what) + " is refused");
    };
    const auto bad = [&](auto args, auto change) {
        change(args);
        return args;
    };
    using enum hb::ErrorCode;
    refused(Unsupported, "codes of quantized values", [&] { be.quantize_rows(st, bad(qx, [](auto& a) { a.type = hb::DType::Q8_0; })); });
    refused(Config, "an unknown variant", [&] { be.quantize_rows(st, bad(qx, [](auto& a) { a.kernel.variant_id = 58; })); });
    refused(Kernel, "scales too short", [&] { be.quantize_rows(st, bad(qx, [](auto& a) { a.scales.bytes = 4; })); });
    refused(Kernel, "codes over x", [&] { be.quantize_rows(st, bad(qx, [&](auto& a) { a.codes = of(x); })); });
    refused(Kernel, "codes without their padding", [&] { be.gemm_i8(st, bad(ga, [](auto& a) { a.x.bytes = kRows * kIn; })); });
    refused(Kernel, "y too short", [&] { be.gemm_i8(st, bad(ga, [](auto& a) { a.n_vec = kRows + 1; })); });
    refused(Kernel, "a code stride of 200", [&] { be.gemm_i8(st, bad(ga, [](auto& a) { a.w.row_stride = kIn; })); });
    refused(Config, "another op's variant", [&] { be.gemm_i8(st, bad(ga, [](auto& a) { a.kernel.variant_id = 57; })); });
    refused(Unsupported, "three parts", [&] { be.norm_rope(st, bad(na, [](auto& a) { a.rope.n_parts = 3; })); });
    refused(Kernel, "a negative eps", [&] { be.norm_rope(st, bad(na, [](auto& a) { a.eps = -1.0f; })); });
    refused(Kernel, "weights too short", [&] { be.norm_rope(st, bad(na, [](auto& a) { a.norm_w[1].bytes = 4 * (kDim - 1); })); });
    refused(Unsupported, "a k_dim of 80", [&] { be.linear_attention(st, bad(la, [](auto& a) { a.k_dim = 80; })); });
    refused(Kernel, "a pool too small", [&] { be.linear_attention(st, bad(la, [](auto& a) { a.n_slots = kSlots + 1; })); });
    refused(Kernel, "states with a stride", [&] { be.linear_attention(st, bad(la, [](auto& a) { a.state.row_stride = 8; })); });
    refused(Kernel, "out over q", [&] { be.linear_attention(st, bad(la, [&](auto& a) { a.out = a.q; })); });
    refused(Kernel, "too few row_starts", [&] { be.linear_attention(st, bad(la, [](auto& a) { a.n_seqs = 3; })); });
    const std::vector<std::byte> image(state->bytes());
    auto frozen = be.import_host_readonly(image);
    refused(Kernel, "read-only states", [&] { be.linear_attention(st, bad(la, [&](auto& a) { a.state = of(frozen); })); });

    // what the device finds is reported by wait(), or left in the caller's word
    auto wrong = dev.up(std::vector<int32_t>{2, 2});
    la.slots = of(wrong);
    be.linear_attention(st, la);
    refused(Kernel, "a slot twice", [&] { st.wait(); });
    check(code_of([&] { st.wait(); }) == -1, "the status is reported once");
    auto word = dev.up(std::vector<uint32_t>{0xFFu});
    la.status = of(word);
    be.linear_attention(st, la);
    check(code_of([&] { st.wait(); }) == -1 && dev.down<uint32_t>(*word)[0] == hb::kStatusBadIndex, "a status word of the caller's");
}

}  // namespace

int main(int argc, char** argv) {
    if (argc > 1 && std::strcmp(argv[1], "--list") == 0) {
        std::printf("backend_layer\n");
        return 0;
    }
    try {
        auto be = hb::make_mi355x_backend(0);
        auto st = be->create_stream();
        const std::pair<hb::OpId, uint32_t> ids[] = {{hb::OpId::NormRope, 56}, {hb::OpId::QuantizeRows, 57}, {hb::OpId::GemmI8, 58}, {hb::OpId::LinearAttention, 59}};
        for (const auto& [op, id] : ids) check(be->variants(op).size() == 1 && be->variants(op)[0].id == id, "the variants' ids are pinned");
        layer(*be, *st);
    } catch (const std::exception& e) {
        std::printf("FAIL exception: %s\n", e.what());
        ++g_failures;
    }
    std::printf("backend_layer: %d checks, %d failures\n", g_checks, g_failures);
    return g_failures ? 1 : 0;
}
