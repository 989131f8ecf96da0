// Stand-alone check of the C ABI from plain C++: no torch, no Python.  Loads the shared library given
// on the command line, allocates with hipMalloc, and verifies known answers bit for bit:
//   hyena_mr_fwd / hyena_fir_cl_fwd   impulse response with bf16-exact taps equals the filter
//   hyena_fir_layer_fwd_rows          the same impulse response behind a featurizer that delays by two samples
//   hyena_li_layer_fwd                with identity featurizer taps equals hyena_li_fwd, outputs and state
//   hyena_fir_step                    dot product over a ring cache, slot rotation
//   hyena_fir_step_far                the same step on a deep cache read whole only every third token, 3 ring periods
//   hyena_iir_step                    one modal update against the closed form
//   hyena_iir_step_win                the modal step with the state in windows of tokens against hyena_iir_step (float32 rounding)
//   hyena_rotary_append, hyena_attn_step, hyena_kv_copy_pages
//                                     a quarter turn written into a page, equal scores give the mean value, a page copied
//   argument errors                   negative return codes and a message
// Usage: abi_selftest /path/to/libhyena_mi355x.so
#include <dlfcn.h>
#include <math.h>
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <vector>

#include "../../include/hyena_mi355x.h"

#define HIP_OK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { printf("HIP error %s at line %d\n", hipGetErrorString(e_), __LINE__); exit(2); } } while (0)
#define CHECK(c, ...) do { if (!(c)) { printf("FAILED line %d: ", __LINE__); printf(__VA_ARGS__); printf("\n"); exit(1); } } while (0)

static uint16_t to_bf16(float f) {           // round to nearest even
    uint32_t u; memcpy(&u, &f, 4);
    u += 0x7fffu + ((u >> 16) & 1u);
    return (uint16_t)(u >> 16);
}
static float from_bf16(uint16_t h) { uint32_t u = (uint32_t)h << 16; float f; memcpy(&f, &u, 4); return f; }

template <class T> static T* dev(const std::vector<T>& v) {
    T* p; HIP_OK(hipMalloc(&p, v.size() * sizeof(T) + 16));
    HIP_OK(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice));
    return p;
}
template <class T> static std::vector<T> host(const T* p, size_t n) {
    std::vector<T> v(n); HIP_OK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost)); return v;
}

int main(int argc, char** argv) {
    if (argc < 2) { printf("usage: %s libhyena_mi355x.so\n", argv[0]); return 2; }
    void* lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) { printf("dlopen failed: %s\n", dlerror()); return 2; }
#define SYM(name) auto p_##name = (decltype(&name))dlsym(lib, #name); CHECK(p_##name, "missing symbol " #name);
    SYM(hyena_version) SYM(hyena_last_error_string) SYM(hyena_mr_fwd) SYM(hyena_fir_cl_fwd) SYM(hyena_fir_step)
    SYM(hyena_iir_step) SYM(hyena_se_fwd) SYM(hyena_fir_step_dpos) SYM(hyena_ring_advance)
    SYM(hyena_fir_step_far) SYM(hyena_fir_far_period) SYM(hyena_fir_far_bytes)
    SYM(hyena_iir_step_win) SYM(hyena_iir_window_flush) SYM(hyena_iir_window_tokens) SYM(hyena_iir_window_supported)
    SYM(hyena_fir_layer_fwd_rows) SYM(hyena_li_layer_fwd) SYM(hyena_li_fwd) SYM(hyena_li_plan) SYM(hyena_li_plan_bytes)
    SYM(hyena_set_launch_override)
    SYM(hyena_rotary_append) SYM(hyena_attn_step) SYM(hyena_attn_step_ws_bytes) SYM(hyena_kv_copy_pages)
    printf("%s\n", p_hyena_version());
    hipStream_t stream; HIP_OK(hipStreamCreate(&stream));

    // ---- impulse responses: B=1, D=32 (2 groups of 16), K=128, bf16-exact taps
    const int64_t B = 1, D = 32, L = 1024, G = 2; const int K = 128;
    std::vector<float> h(G * K);
    for (int g = 0; g < G; ++g) for (int k = 0; k < K; ++k) h[g * K + k] = (float)((k * 5 + g * 3) % 17 - 8) / 16.f;
    const int pos[2] = {300, 511};
    std::vector<uint16_t> one(B * D * L, to_bf16(1.f)), imp(B * D * L, 0), imp_cl(B * L * D, 0);
    for (int d = 0; d < D; ++d) for (int p : pos) { imp[d * L + p] = to_bf16(1.f); imp_cl[p * D + d] = to_bf16(1.f); }
    float* dh = dev(h);
    uint16_t *d_one = dev(one), *d_imp = dev(imp), *d_impcl = dev(imp_cl), *d_out;
    HIP_OK(hipMalloc(&d_out, B * D * L * 2));
    {
        hyena_rows r1 = {d_imp, D * L, L, D, D}, r2 = {d_one, D * L, L, D, D};
        int rc = p_hyena_mr_fwd(&r1, &r2, &r2, dh, 0, nullptr, HYENA_BIAS_NONE, d_out, B, D, L, G, K, stream);
        CHECK(rc == 0, "hyena_mr_fwd rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto o = host(d_out, (size_t)(B * D * L));
        for (int d = 0; d < D; ++d) for (int t = 0; t < L; ++t) {
            float e = 0.f;
            for (int p : pos) if (t >= p && t - p < K) e += h[(d / 16) * K + t - p];
            CHECK(from_bf16(o[d * L + t]) == from_bf16(to_bf16(e)), "hyena_mr_fwd d=%d t=%d got %g want %g", d, t,
                  from_bf16(o[d * L + t]), e);
        }
        printf("hyena_mr_fwd impulse response: ok\n");
    }
    {
        hyena_cl c1 = {d_impcl, L * D, D}, c2 = {d_one, L * D, D};
        int rc = p_hyena_fir_cl_fwd(&c1, &c2, &c2, dh, 0, nullptr, HYENA_BIAS_NONE, d_out, nullptr, nullptr, 0, B, L, D, G,
                                    K, stream);
        CHECK(rc == 0, "hyena_fir_cl_fwd rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto o = host(d_out, (size_t)(B * D * L));
        for (int d = 0; d < D; ++d) for (int t = 0; t < L; ++t) {
            float e = 0.f;
            for (int p : pos) if (t >= p && t - p < K) e += h[(d / 16) * K + t - p];
            CHECK(from_bf16(o[t * D + d]) == from_bf16(to_bf16(e)), "hyena_fir_cl_fwd d=%d t=%d got %g want %g", d, t,
                  from_bf16(o[t * D + d]), e);
        }
        printf("hyena_fir_cl_fwd impulse response: ok\n");
    }

    // ---- a layer from a sequence-major projection p [B][3D][L] (plain split: rows x2 | x1 | v).  Featurizer taps:
    // x1 (1, 0, 0) = a delay of two samples, x2 (0.5, 0.25, 0.25) = 1 from t = 2 on for a row of ones, v (0, 0, 1) = the
    // identity.  The x1 rows hold the impulses, so the output is the filter's impulse response two samples late.
    {
        std::vector<uint16_t> proj(B * 3 * D * L, to_bf16(1.f));
        for (int d = 0; d < D; ++d) for (int t = 0; t < L; ++t) proj[(D + d) * L + t] = imp[d * L + t];
        std::vector<float> ft(3 * D * 3, 0.f);
        for (int d = 0; d < D; ++d) {
            ft[(0 * D + d) * 3 + 0] = 1.f;
            ft[(1 * D + d) * 3 + 0] = 0.5f; ft[(1 * D + d) * 3 + 1] = 0.25f; ft[(1 * D + d) * 3 + 2] = 0.25f;
            ft[(2 * D + d) * 3 + 2] = 1.f;
        }
        uint16_t* d_p = dev(proj); float* d_ft = dev(ft);
        hyena_rows q2 = {d_p, 3 * D * L, L, D, D}, q1 = {d_p + D * L, 3 * D * L, L, D, D}, qv = {d_p + 2 * D * L, 3 * D * L, L, D, D};
        int rc = p_hyena_fir_layer_fwd_rows(&q1, &q2, &qv, d_ft, 3, dh, 0, nullptr, HYENA_BIAS_NONE, d_out, B, D, L, G, K, stream);
        CHECK(rc == 0, "hyena_fir_layer_fwd_rows rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto o = host(d_out, (size_t)(B * D * L));
        for (int d = 0; d < D; ++d) for (int t = 0; t < L; ++t) {
            float e = 0.f;
            for (int pp : pos) if (t - 2 >= pp && t - 2 - pp < K) e += h[(d / 16) * K + t - 2 - pp];
            CHECK(from_bf16(o[d * L + t]) == from_bf16(to_bf16(e)), "hyena_fir_layer_fwd_rows d=%d t=%d got %g want %g", d, t,
                  from_bf16(o[d * L + t]), e);
        }
        printf("hyena_fir_layer_fwd_rows impulse response behind a two-sample featurizer delay: ok\n");

        // the same projection through hyena_li_layer_fwd with identity featurizer taps on every row must be
        // hyena_li_fwd on the rows themselves, bit for bit (lone wavefronts on both sides)
        const int64_t S = 16;
        std::vector<float> lp(G * S * 2, 0.f), rs(G * S * 2, 0.f);
        for (int g = 0; g < G; ++g) for (int m = 0; m < S; ++m) {
            lp[(g * S + m) * 2] = -0.02f * (float)(m + 1 + g);  lp[(g * S + m) * 2 + 1] = 0.1f * (float)m;
            rs[(g * S + m) * 2] = 0.25f - 0.03f * (float)m;     rs[(g * S + m) * 2 + 1] = 0.01f * (float)(m + g);
        }
        std::vector<float> idt(3 * D * 3, 0.f);
        for (int i = 0; i < 3 * D; ++i) idt[i * 3 + 2] = 1.f;
        for (int d = 0; d < D; ++d) for (int t = 0; t < L; ++t) {               // less trivial gates than ones
            proj[d * L + t] = to_bf16((float)((t * 7 + d) % 13 - 6) / 8.f);
            proj[(2 * D + d) * L + t] = to_bf16((float)((t * 3 + d * 5) % 11 - 5) / 4.f);
            proj[(D + d) * L + t] = to_bf16((float)((t + d * 2) % 9 - 4) / 4.f);
        }
        HIP_OK(hipMemcpy(d_p, proj.data(), proj.size() * 2, hipMemcpyHostToDevice));
        float *d_lp = dev(lp), *d_rs = dev(rs), *d_id = dev(idt), *d_st0, *d_st1; void* d_ws; uint16_t* d_out2;
        HIP_OK(hipMalloc(&d_ws, (size_t)p_hyena_li_plan_bytes(G, S)));
        HIP_OK(hipMalloc(&d_out2, B * D * L * 2));
        HIP_OK(hipMalloc(&d_st0, B * D * S * 2 * 4)); HIP_OK(hipMalloc(&d_st1, B * D * S * 2 * 4));
        rc = p_hyena_li_plan(d_lp, d_rs, G, S, d_ws, stream);
        CHECK(rc == 0, "hyena_li_plan rc=%d: %s", rc, p_hyena_last_error_string());
        // (the same work decomposition on both sides: the order of the scan's additions depends on it)
        CHECK(p_hyena_set_launch_override("li_coop", 0) == 0, "li_coop override");
        CHECK(p_hyena_set_launch_override("li_cpw", 4) == 0, "li_cpw override");
        rc = p_hyena_li_fwd(&q1, &q2, &qv, d_ws, nullptr, 1, d_out, nullptr, d_st0, B, D, L, G, S, stream);
        CHECK(rc == 0, "hyena_li_fwd rc=%d: %s", rc, p_hyena_last_error_string());
        rc = p_hyena_li_layer_fwd(&q1, &q2, &qv, d_id, 3, d_ws, nullptr, 1, d_out2, d_st1, B, D, L, G, S, stream);
        CHECK(rc == 0, "hyena_li_layer_fwd rc=%d: %s", rc, p_hyena_last_error_string());
        CHECK(p_hyena_set_launch_override("li_coop", -1) == 0, "li_coop override reset");
        CHECK(p_hyena_set_launch_override("li_cpw", -1) == 0, "li_cpw override reset");
        HIP_OK(hipStreamSynchronize(stream));
        auto oa = host(d_out, (size_t)(B * D * L)); auto ob = host(d_out2, (size_t)(B * D * L));
        CHECK(oa == ob, "hyena_li_layer_fwd with identity featurizer taps differs from hyena_li_fwd");
        auto sa = host(d_st0, (size_t)(B * D * S * 2)); auto sb = host(d_st1, (size_t)(B * D * S * 2));
        CHECK(memcmp(sa.data(), sb.data(), sa.size() * 4) == 0, "hyena_li_layer_fwd state differs from hyena_li_fwd");
        bool nonzero = false;
        for (auto x : ob) nonzero |= (x & 0x7fff) != 0;
        CHECK(nonzero, "hyena_li_layer_fwd wrote only zeros");
        printf("hyena_li_layer_fwd with identity featurizer taps equals hyena_li_fwd (outputs and state): ok\n");
    }

    // ---- decode FIR step: ring [B=2][R=6][D=16], per-channel taps, two steps (slot rotation)
    {
        const int64_t Bs = 2, Ds = 16, R = 6;
        std::vector<uint16_t> ring(Bs * R * Ds), u(Bs * Ds), one_s(Bs * Ds, to_bf16(1.f));
        std::vector<float> w(Ds * (R + 1));
        for (size_t i = 0; i < ring.size(); ++i) ring[i] = to_bf16((float)((int)(i % 11) - 5) / 4.f);
        for (size_t i = 0; i < u.size(); ++i) u[i] = to_bf16((float)((int)(i % 7) - 3) / 2.f);
        for (size_t i = 0; i < w.size(); ++i) w[i] = (float)((int)(i % 5) - 2) / 8.f;
        uint16_t *d_ring = dev(ring), *d_u = dev(u), *d_1 = dev(one_s), *d_y; float* d_w = dev(w);
        HIP_OK(hipMalloc(&d_y, Bs * Ds * 2));
        std::vector<uint16_t> hist = ring;      // host model of the ring contents
        for (int step = 0; step < 2; ++step) {
            const int64_t p = step;             // oldest slot
            int rc = p_hyena_fir_step(d_u, d_1, d_1, Ds, d_ring, R, Ds, p, d_w, nullptr, HYENA_BIAS_NONE, d_y, Ds, Bs, Ds, Ds, stream);
            CHECK(rc == 0, "hyena_fir_step rc=%d: %s", rc, p_hyena_last_error_string());
            HIP_OK(hipStreamSynchronize(stream));
            auto y = host(d_y, (size_t)(Bs * Ds));
            for (int b = 0; b < Bs; ++b) for (int d = 0; d < Ds; ++d) {
                float acc = 0.f;
                for (int i = 0; i < R; ++i) acc += w[d * (R + 1) + i] * from_bf16(hist[(b * R + (p + i) % R) * Ds + d]);
                acc += w[d * (R + 1) + R] * from_bf16(u[b * Ds + d]);
                CHECK(from_bf16(y[b * Ds + d]) == from_bf16(to_bf16(acc)), "hyena_fir_step step %d b=%d d=%d got %g want %g",
                      step, b, d, from_bf16(y[b * Ds + d]), acc);
            }
            for (int b = 0; b < Bs; ++b) for (int d = 0; d < Ds; ++d) hist[(b * R + p) * Ds + d] = u[b * Ds + d];
            auto rr = host(d_ring, ring.size());
            CHECK(rr == hist, "hyena_fir_step ring contents after step %d", step);
        }
        printf("hyena_fir_step on a ring cache: ok\n");

        // the same ring continued with its position in device memory: seven more steps, so the ring wraps
        std::vector<int32_t> pos_h = {2, 0}, depth_h = {(int32_t)R, 5};     // a second, unused ring of depth 5
        int32_t *d_pos = dev(pos_h), *d_depth = dev(depth_h);
        for (int step = 2; step < 9; ++step) {
            const int64_t p = step % R;
            for (size_t i = 0; i < u.size(); ++i) u[i] = to_bf16((float)((int)((i + 3 * step) % 9) - 4) / 2.f);
            HIP_OK(hipMemcpy(d_u, u.data(), u.size() * 2, hipMemcpyHostToDevice));
            int rc = p_hyena_fir_step_dpos(d_u, d_1, d_1, Ds, d_ring, R, Ds, d_pos, d_w, nullptr, HYENA_BIAS_NONE, d_y, Ds, Bs, Ds, Ds, stream);
            CHECK(rc == 0, "hyena_fir_step_dpos rc=%d: %s", rc, p_hyena_last_error_string());
            rc = p_hyena_ring_advance(d_pos, d_depth, 2, stream);
            CHECK(rc == 0, "hyena_ring_advance rc=%d: %s", rc, p_hyena_last_error_string());
            HIP_OK(hipStreamSynchronize(stream));
            auto y = host(d_y, (size_t)(Bs * Ds));
            for (int b = 0; b < Bs; ++b) for (int d = 0; d < Ds; ++d) {
                float acc = 0.f;
                for (int i = 0; i < R; ++i) acc += w[d * (R + 1) + i] * from_bf16(hist[(b * R + (p + i) % R) * Ds + d]);
                acc += w[d * (R + 1) + R] * from_bf16(u[b * Ds + d]);
                CHECK(from_bf16(y[b * Ds + d]) == from_bf16(to_bf16(acc)), "hyena_fir_step_dpos step %d b=%d d=%d got %g want %g",
                      step, b, d, from_bf16(y[b * Ds + d]), acc);
            }
            for (int b = 0; b < Bs; ++b) for (int d = 0; d < Ds; ++d) hist[(b * R + p) * Ds + d] = u[b * Ds + d];
            CHECK(host(d_ring, ring.size()) == hist, "hyena_fir_step_dpos ring contents after step %d", step);
            auto ph = host(d_pos, 2);
            CHECK(ph[0] == (step + 1) % R && ph[1] == (step - 1) % 5, "hyena_ring_advance positions after step %d: %d %d", step, ph[0], ph[1]);
        }
        printf("hyena_fir_step_dpos / hyena_ring_advance (positions in device memory): ok\n");
    }

    // ---- decode FIR step with far sums: ring [B=3][D/512=2][R=40][512] in channel blocks, taps shared by groups of
    // 16 channels; small dyadic values, so every float32 sum is exact whatever its order and the outputs must be equal
    // bit for bit to the host model for three periods of the ring
    {
        const int64_t Bs = 3, Ds = 1024, R = 40, Gs = Ds / 16, cb = 512;
        const int64_t period = p_hyena_fir_far_period(R);
        CHECK(period % R == 0 && period / R == p_hyena_fir_far_period(1) && period / R >= 2, "far period %lld", (long long)period);
        std::vector<uint16_t> ring(Bs * R * Ds), u(Bs * Ds), one_s(Bs * Ds, to_bf16(1.f));
        std::vector<float> w(Gs * (R + 1));
        auto slot = [&](int64_t b, int64_t s, int64_t d) { return ((b * (Ds / cb) + d / cb) * R + s) * cb + d % cb; };
        std::vector<float> hist(Bs * R * Ds);                       // hist[(b*R + i)*Ds + d]: i-th oldest sample
        for (int64_t b = 0; b < Bs; ++b) for (int64_t i = 0; i < R; ++i) for (int64_t d = 0; d < Ds; ++d) {
            const float val = (float)((int)((b * 7 + i * 3 + d) % 9) - 4) / 4.f;
            hist[(b * R + i) * Ds + d] = val;
            ring[slot(b, i, d)] = to_bf16(val);                     // counter 0: slot i is the i-th oldest
        }
        for (size_t i = 0; i < w.size(); ++i) w[i] = (float)((int)(i % 7) - 3) / 8.f;
        uint16_t *d_ring = dev(ring), *d_u = dev(u), *d_1 = dev(one_s), *d_y; float *d_w = dev(w), *d_far;
        HIP_OK(hipMalloc(&d_y, Bs * Ds * 2));
        HIP_OK(hipMalloc(&d_far, (size_t)p_hyena_fir_far_bytes(Bs, Ds)));
        for (int step = 0; step < 3 * R + 2; ++step) {
            for (size_t i = 0; i < u.size(); ++i) u[i] = to_bf16((float)((int)((i + 5 * step) % 9) - 4) / 2.f);
            HIP_OK(hipMemcpy(d_u, u.data(), u.size() * 2, hipMemcpyHostToDevice));
            const int64_t cnt = step % period;
            int rc = p_hyena_fir_step_far(d_u, d_1, d_1, Ds, d_ring, R, cb, cnt, nullptr, d_far, step == 0, d_w, nullptr,
                                          HYENA_BIAS_NONE, d_y, Ds, Bs, Ds, Gs, stream);
            CHECK(rc == 0, "hyena_fir_step_far rc=%d: %s", rc, p_hyena_last_error_string());
            HIP_OK(hipStreamSynchronize(stream));
            auto y = host(d_y, (size_t)(Bs * Ds));
            for (int64_t b = 0; b < Bs; ++b) for (int64_t d = 0; d < Ds; ++d) {
                float acc = 0.f;
                for (int64_t i = 0; i < R; ++i) acc += w[(d / 16) * (R + 1) + i] * hist[(b * R + i) * Ds + d];
                acc += w[(d / 16) * (R + 1) + R] * from_bf16(u[b * Ds + d]);
                CHECK(from_bf16(y[b * Ds + d]) == from_bf16(to_bf16(acc)), "hyena_fir_step_far step %d b=%lld d=%lld got %g want %g",
                      step, (long long)b, (long long)d, from_bf16(y[b * Ds + d]), acc);
            }
            for (int64_t b = 0; b < Bs; ++b) for (int64_t d = 0; d < Ds; ++d) {          // the window moves on by one sample
                for (int64_t i = 0; i + 1 < R; ++i) hist[(b * R + i) * Ds + d] = hist[(b * R + i + 1) * Ds + d];
                hist[(b * R + R - 1) * Ds + d] = from_bf16(u[b * Ds + d]);
            }
        }
        auto rr = host(d_ring, ring.size());
        const int64_t pos_end = (3 * R + 2) % R;
        for (int64_t b = 0; b < Bs; ++b) for (int64_t i = 0; i < R; ++i) for (int64_t d = 0; d < Ds; d += 37)
            CHECK(from_bf16(rr[slot(b, (pos_end + i) % R, d)]) == hist[(b * R + i) * Ds + d], "hyena_fir_step_far ring contents");
        printf("hyena_fir_step_far (channel-blocked cache, windows of %lld tokens): ok\n", (long long)(period / R));
    }

    // ---- decode IIR step, real poles: state = p*state + x1v ; y = x2 * (sum r*state + D*x1v)
    {
        const int64_t Bs = 2, Ds = 8, S = 16;
        std::vector<float> st(Bs * Ds * S), poles(Ds * S), res(Ds * S), Dc(Ds);
        std::vector<uint16_t> x1(Bs * Ds), x2(Bs * Ds), v(Bs * Ds);
        for (size_t i = 0; i < st.size(); ++i) st[i] = (float)((int)(i % 9) - 4) / 4.f;
        for (size_t i = 0; i < poles.size(); ++i) { poles[i] = 0.5f + (float)(i % 4) / 8.f; res[i] = (float)((int)(i % 3) - 1) / 2.f; }
        for (int d = 0; d < Ds; ++d) Dc[d] = (float)(d - 4) / 4.f;
        for (size_t i = 0; i < x1.size(); ++i) { x1[i] = to_bf16((float)((int)(i % 5) - 2)); x2[i] = to_bf16((float)((int)(i % 3) + 1)); v[i] = to_bf16(0.5f); }
        float *d_st = dev(st), *d_p = dev(poles), *d_r = dev(res), *d_D = dev(Dc), *d_y;
        uint16_t *d1 = dev(x1), *d2 = dev(x2), *dv = dev(v);
        HIP_OK(hipMalloc(&d_y, Bs * Ds * 4));
        int rc = p_hyena_iir_step(d1, d2, dv, Ds, d_st, d_p, d_r, 0, d_D, 0, d_y, 1, Ds, Bs, Ds, Ds, S, stream);
        CHECK(rc == 0, "hyena_iir_step rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto y = host(d_y, (size_t)(Bs * Ds)); auto ns = host(d_st, st.size());
        for (int b = 0; b < Bs; ++b) for (int d = 0; d < Ds; ++d) {
            const float x1v = from_bf16(to_bf16(from_bf16(x1[b * Ds + d]) * from_bf16(v[b * Ds + d])));
            double sum = 0.0;
            for (int s = 0; s < S; ++s) {
                const float e = poles[d * S + s] * st[(b * Ds + d) * S + s] + x1v;     // exact in fp32 for these values
                CHECK(ns[(b * Ds + d) * S + s] == e, "hyena_iir_step state b=%d d=%d s=%d", b, d, s);
                sum += (double)res[d * S + s] * e;
            }
            const float want = from_bf16(x2[b * Ds + d]) * ((float)sum + Dc[d] * x1v);
            CHECK(fabsf(y[b * Ds + d] - want) <= 1e-5f * (1.f + fabsf(want)), "hyena_iir_step y b=%d d=%d got %g want %g", b, d,
                  y[b * Ds + d], want);
        }
        printf("hyena_iir_step closed form: ok\n");
    }

    // ---- windowed modal step from C: the caller owns hist / far / g, counts tokens and warm; against hyena_iir_step on a
    //      copy of the state, outputs on every token and the state after a flush
    {
        const int64_t Bs = 16, Ds = 4096, S = 16, W = p_hyena_iir_window_tokens();
        CHECK(p_hyena_iir_window_supported(Bs, Ds, S, 0) == 1, "windowed step not offered for B=16 D=4096");
        std::vector<float> st(Bs * Ds * S), poles(Ds * S), res(Ds * S), Dc(Ds), g(Ds * W);
        uint32_t rng = 12345u;
        auto rnd = [&]() { rng = rng * 1664525u + 1013904223u; return (float)((rng >> 8) & 0xffff) / 65536.f - 0.5f; };
        for (auto& x : st) x = rnd();
        for (auto& x : poles) x = 0.5f + 0.9f * rnd();           // 0.05 .. 0.95
        for (auto& x : res) x = rnd();
        for (auto& x : Dc) x = rnd();
        for (int64_t d = 0; d < Ds; ++d) for (int64_t k = 0; k < W; ++k) {
            double acc = 0.0;
            for (int64_t s = 0; s < S; ++s) acc += (double)res[d * S + s] * pow((double)poles[d * S + s], (double)k);
            g[d * W + k] = (float)acc;
        }
        float *d_sa = dev(st), *d_sb = dev(st), *d_p = dev(poles), *d_r = dev(res), *d_D = dev(Dc), *d_g = dev(g), *d_ya, *d_yb, *d_far;
        uint16_t* d_hist;
        HIP_OK(hipMalloc(&d_ya, Bs * Ds * 4)); HIP_OK(hipMalloc(&d_yb, Bs * Ds * 4));
        HIP_OK(hipMalloc(&d_far, Bs * W * Ds * 4)); HIP_OK(hipMalloc(&d_hist, Bs * W * Ds * 2));
        HIP_OK(hipMemset(d_far, 0, Bs * W * Ds * 4)); HIP_OK(hipMemset(d_hist, 0, Bs * W * Ds * 2));
        std::vector<uint16_t> x1(Bs * Ds), x2(Bs * Ds), v(Bs * Ds);
        uint16_t *d1 = dev(x1), *d2 = dev(x2), *dv = dev(v);
        hyena_iir_window win = {};
        win.hist = d_hist; win.far = d_far; win.g = d_g;
        int warm = 0;
        auto flush_and_compare = [&](int step) {          // step = tokens done so far - 1; the flush takes the next token's counter
            win.cnt = (step + 1) % W; win.warm = warm;
            int rc = p_hyena_iir_window_flush(d_sa, d_p, d_r, 0, Bs, Ds, Ds, S, &win, stream);
            CHECK(rc == 0, "hyena_iir_window_flush rc=%d: %s", rc, p_hyena_last_error_string());
            warm = 0;
            HIP_OK(hipStreamSynchronize(stream));
            auto sa = host(d_sa, st.size()); auto sb = host(d_sb, st.size());
            for (size_t i = 0; i < sa.size(); ++i)
                CHECK(fabsf(sa[i] - sb[i]) <= 3e-5f * (1.f + fabsf(sb[i])), "windowed state after flush, step %d i=%zu got %g want %g",
                      step, i, sa[i], sb[i]);
        };
        for (int step = 0; step < 11; ++step) {
            for (auto& x : x1) x = to_bf16(rnd());
            for (auto& x : x2) x = to_bf16(1.f + rnd());
            for (auto& x : v) x = to_bf16(2.f * rnd());
            HIP_OK(hipMemcpy(d1, x1.data(), x1.size() * 2, hipMemcpyHostToDevice));
            HIP_OK(hipMemcpy(d2, x2.data(), x2.size() * 2, hipMemcpyHostToDevice));
            HIP_OK(hipMemcpy(dv, v.data(), v.size() * 2, hipMemcpyHostToDevice));
            win.cnt = step % W; win.warm = warm;
            int rc = p_hyena_iir_step_win(d1, d2, dv, Ds, d_sa, d_p, d_r, 0, d_D, 0, d_ya, 1, Ds, Bs, Ds, Ds, S, &win, stream);
            CHECK(rc == 0, "hyena_iir_step_win rc=%d: %s", rc, p_hyena_last_error_string());
            warm = warm < W ? warm + 1 : (int)W;
            rc = p_hyena_iir_step(d1, d2, dv, Ds, d_sb, d_p, d_r, 0, d_D, 0, d_yb, 1, Ds, Bs, Ds, Ds, S, stream);
            CHECK(rc == 0, "hyena_iir_step rc=%d: %s", rc, p_hyena_last_error_string());
            HIP_OK(hipStreamSynchronize(stream));
            auto ya = host(d_ya, (size_t)(Bs * Ds)); auto yb = host(d_yb, (size_t)(Bs * Ds));
            for (size_t i = 0; i < ya.size(); ++i)
                CHECK(fabsf(ya[i] - yb[i]) <= 1e-4f * (1.f + fabsf(yb[i])), "hyena_iir_step_win step %d i=%zu got %g want %g", step,
                      i, ya[i], yb[i]);
            if (step == 5) flush_and_compare(step);          // in the middle of the windows; they restart
        }
        flush_and_compare(10);
        printf("hyena_iir_step_win / hyena_iir_window_flush (windows of %lld tokens) against hyena_iir_step: ok\n", (long long)W);
    }

    // ---- paged key / value cache: two sequences, pages of 16 positions, 2 query heads on one key head of 64
    {
        const int64_t hd = 64, ps = 16, P = 5, S = 2, H = 2, T = 6;     // three tokens a sequence
        std::vector<uint16_t> q(T * H * hd), k(T * hd), v(T * hd), zero(P * ps * hd, 0);
        for (int64_t t = 0; t < T; ++t)
            for (int64_t d = 0; d < hd; ++d) {
                k[t * hd + d] = to_bf16((float)(t + 1) * (d < 32 ? 1.f : 0.5f));
                v[t * hd + d] = to_bf16((float)(4 * t + d % 4));
                for (int64_t h = 0; h < H; ++h) q[(t * H + h) * hd + d] = to_bf16(d < 32 ? 2.f : -1.f);
            }
        std::vector<int32_t> table = {3, 1, 4, -1}, pos = {14, 15, 16, 0, 1, 2}, lens = {17, 3};
        std::vector<double> turns(hd / 2, 0.25);                        // position p: p quarter turns
        uint16_t *dq = dev(q), *dk = dev(k), *dv = dev(v), *kp = dev(zero), *vp = dev(zero), *qo = dev(q), *out = dev(q);
        int32_t *d_table = dev(table), *d_pos = dev(pos), *d_lens = dev(lens);
        double* d_turns = dev(turns);
        hyena_kv_pages kv = {};
        kv.k = {kp, ps * hd, ps * hd, hd, nullptr};
        kv.v = {vp, ps * hd, ps * hd, hd, nullptr};
        kv.num_pages = P, kv.page_size = ps, kv.kv_heads = 1, kv.head_dim = hd;
        kv.table = d_table, kv.table_stride = 2, kv.table_width = 2, kv.sequences = S, kv.dtype = HYENA_DTYPE_BF16;
        hyena_heads hq = {dq, H * hd, hd}, hk = {dk, hd, hd}, hv = {dv, hd, hd}, ho = {qo, H * hd, hd};
        int rc = p_hyena_rotary_append(&kv, &hq, &hk, &hv, &ho, nullptr, d_pos, nullptr, d_turns, hd, 0, 0, T, H,
                                       HYENA_DTYPE_BF16, stream);
        CHECK(rc == 0, "hyena_rotary_append rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto pk = host(kp, zero.size()); auto pv = host(vp, zero.size()); auto pq = host(qo, q.size());
        const int64_t at[6] = {3 * ps + 14, 3 * ps + 15, 1 * ps, 4 * ps, 4 * ps + 1, 4 * ps + 2};
        for (int64_t t = 0; t < T; ++t) {
            const int quarter = pos[t] % 4;
            const float c[4] = {1, 0, -1, 0}, sn[4] = {0, 1, 0, -1};
            for (int64_t d = 0; d < 32; ++d) {
                const float x1 = (float)(t + 1), x2 = 0.5f * (t + 1);
                CHECK(from_bf16(pk[at[t] * hd + d]) == x1 * c[quarter] - x2 * sn[quarter] &&
                          from_bf16(pk[at[t] * hd + 32 + d]) == x1 * sn[quarter] + x2 * c[quarter], "rotated key t=%d d=%d", (int)t, (int)d);
                CHECK(pv[at[t] * hd + d] == v[t * hd + d], "value t=%d d=%d", (int)t, (int)d);
                CHECK(from_bf16(pq[t * H * hd + d]) == 2.f * c[quarter] + sn[quarter], "rotated query t=%d d=%d", (int)t, (int)d);
            }
        }
        // scale 0: every position weighs the same; sequence 0 sees 14 zero values ahead of its three, sequence 1 its three
        const int64_t nws = p_hyena_attn_step_ws_bytes(&kv, H);
        void* ws; HIP_OK(hipMalloc(&ws, nws + 16));
        hyena_heads h2 = {qo, H * hd, hd};
        rc = p_hyena_attn_step(&kv, &h2, d_lens, 0.f, out, ws, nws, H, HYENA_DTYPE_BF16, stream);
        CHECK(rc == 0, "hyena_attn_step rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto o = host(out, (size_t)(S * H * hd));
        for (int64_t s = 0; s < S; ++s)
            for (int64_t i = 0; i < H * hd; ++i) {
                const int64_t d = i % hd;
                const float want = s == 0 ? (float)(12 + 3 * (d % 4)) / 17.f : (float)(48 + 3 * (d % 4)) / 3.f;
                CHECK(fabsf(from_bf16(o[s * H * hd + i]) - want) <= want / 256.f, "mean value s=%d i=%d got %g want %g", (int)s,
                      (int)i, from_bf16(o[s * H * hd + i]), want);
            }
        std::vector<int32_t> src = {3}, dst = {0};
        int32_t *d_src = dev(src), *d_dst = dev(dst);
        hyena_kv_pools pools = {vp, P * ps * hd * 2, ps * hd * 2, P};
        rc = p_hyena_kv_copy_pages(&pools, &pools, 1, ps * hd * 2, d_src, d_dst, 1, stream);
        CHECK(rc == 0, "hyena_kv_copy_pages rc=%d: %s", rc, p_hyena_last_error_string());
        HIP_OK(hipStreamSynchronize(stream));
        auto pc = host(vp, zero.size());
        CHECK(memcmp(pc.data(), pc.data() + 3 * ps * hd, ps * hd * 2) == 0 && memcmp(pc.data() + ps * hd, pv.data() + ps * hd, 4 * ps * hd * 2) == 0,
              "copied page");
        printf("hyena_rotary_append / hyena_attn_step / hyena_kv_copy_pages on pages: ok\n");
    }

    // ---- rejected arguments come back as negative codes with a message, before anything is launched
    {
        hyena_rows r = {d_one, D * L, L, D, D};
        CHECK(p_hyena_mr_fwd(&r, &r, &r, dh, 0, nullptr, 0, d_out, B, D, L, G, 200, stream) == HYENA_ENOSUP, "K=200 accepted");
        CHECK(strlen(p_hyena_last_error_string()) > 0, "empty error message");
        CHECK(p_hyena_se_fwd(nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr, 1, 16, 8, 1, 7, stream) == HYENA_EINVAL, "null x1 accepted");
        CHECK(p_hyena_mr_fwd(&r, &r, &r, dh, 0, nullptr, 0, d_out, B, D, L - 4, G, K, stream) == HYENA_EALIGN, "L %% 8 accepted");
        printf("argument errors: ok\n");
    }
    HIP_OK(hipDeviceSynchronize());
    printf("abi_selftest: ok\n");
    return 0;
}
