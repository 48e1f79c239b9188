// wf_rope.hip -- rotary positions on rows of q and k.
//
// Pair j of a head's first r dims, j < r / 2, is turned by the angle a = pos * freq[j]:
//     y1 = s (x1 cos a - x2 sin a),  y2 = s (x2 cos a + x1 sin a),
// pairs (j, j + r/2) (half layout) or (2j, 2j + 1) (interleaved), s one factor for all; dims >= r pass.
// The angle: positions reach millions of radians, where 32 bits have lost the fraction of a turn, so
// turns = pos * freq / 2pi are formed in 64 bits, the whole turns dropped there, and only the remainder
// in [-1/2, 1/2] goes to 32 bits (2^-25 of a half turn) and to sincospif. x is widened to 32 bits and each
// result rounded once. A call reads and writes every element once and is bound by that.
//
// A workgroup takes kRopeTokens tokens (one in short calls): its threads first put the tokens' cos and sin
// in LDS, one sincos per (token, pair) for all heads, then walk the heads with two 16-byte loads and
// stores an item (VEC pairs). VEC = 1 takes any stride, alignment and r.
// Measured: 16384 tokens, 20 + 5 heads of 128, bf16: 45 us, 4.65 TB/s (a large copy: 4.90); 128 tokens 3.7 us on the
// device, latencies; 4097 tokens, 8 + 2 heads of 96, f32, interleaved 9.3 us.
#include "wf_common.h"
#include "wf_device.h"

namespace wf {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxDim = 512;

struct RopeArgs {
    const void* x[2];
    void* y[2];
    int64_t xt[2], xh[2], yt[2], yh[2];  // strides of a token and of a head, in elements
    int H[2];
    const void* pos;
    int pos64;
    const double* freq;
    int T, D, r;
    float scale;
};

template <int DT>
struct RopeElem;
template <>
struct RopeElem<DT_F32> {
    using T = float;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ T down(float v) { return v; }
};
template <>
struct RopeElem<DT_BF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float up(T v) { return bf2f(v); }
    static __device__ __forceinline__ T down(float v) { return f2bf(v); }
};
template <>
struct RopeElem<DT_F16> {
    using T = uint16_t;
    static __device__ __forceinline__ float up(T v) { return h2f(v); }
    static __device__ __forceinline__ T down(float v) { return f2h(v); }
};

template <class T, int N>
struct __attribute__((aligned(sizeof(T) * N))) RopeVec {
    T v[N];
};

template <int DT, int VEC, bool INTER, int TOK>
__global__ __launch_bounds__(kRopeThreads) void k_rope(RopeArgs a) {
    using E = RopeElem<DT>;
    using V = RopeVec<typename E::T, VEC>;
    __shared__ float2 cs[TOK][kRopeMaxDim / 2];
    const int half = a.r >> 1, t0 = blockIdx.x * TOK, nt = min(TOK, a.T - t0);
    for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
        const int t = i / half, j = i - t * half;
        const double p = a.pos64 ? (double)((const int64_t*)a.pos)[t0 + t] : (double)((const int32_t*)a.pos)[t0 + t];
        const double turns = p * (a.freq[j] * 0.15915494309189533577);  // 1 / 2pi
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        cs[t][j] = make_float2(c * a.scale, s * a.scale);
    }
    __syncthreads();
    // items of a head: VEC pairs each, then VEC passing dims each
    const int np = half / VEC, per = np + (a.D - a.r) / VEC, HT = a.H[0] + a.H[1];
    for (int i = threadIdx.x; i < nt * HT * per; i += kRopeThreads) {
        const int c = i % per, th = i / per, t = th / HT;
        int h = th - t * HT;
        const int w = h >= a.H[0];
        if (w) h -= a.H[0];
        const typename E::T* x = (const typename E::T*)a.x[w] + (t0 + t) * a.xt[w] + h * a.xh[w];
        typename E::T* y = (typename E::T*)a.y[w] + (t0 + t) * a.yt[w] + h * a.yh[w];
        if (c >= np) {
            const int d = a.r + (c - np) * VEC;
            *reinterpret_cast<V*>(y + d) = *reinterpret_cast<const V*>(x + d);
            continue;
        }
        // the item's two vectors: dims [d0, +VEC) and [d1, +VEC)
        const int d0 = INTER ? 2 * VEC * c : VEC * c, d1 = INTER ? d0 + VEC : d0 + half;
        const V u = *reinterpret_cast<const V*>(x + d0), v = *reinterpret_cast<const V*>(x + d1);
        V yu, yv;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float2 k = cs[t][VEC * c + e];
            // element 2e of the 2 VEC in order (interleaved) or (u[e], v[e])
            const float x1 = E::up(INTER ? (2 * e < VEC ? u.v[2 * e] : v.v[2 * e - VEC]) : u.v[e]);
            const float x2 = E::up(INTER ? (2 * e + 1 < VEC ? u.v[2 * e + 1] : v.v[2 * e + 1 - VEC]) : v.v[e]);
            const typename E::T y1 = E::down(fmaf(x1, k.x, -(x2 * k.y))), y2 = E::down(fmaf(x2, k.x, x1 * k.y));
            if constexpr (INTER) {
                (2 * e < VEC ? yu.v[2 * e] : yv.v[2 * e - VEC]) = y1;
                (2 * e + 1 < VEC ? yu.v[2 * e + 1] : yv.v[2 * e + 1 - VEC]) = y2;
            } else {
                yu.v[e] = y1;
                yv.v[e] = y2;
            }
        }
        *reinterpret_cast<V*>(y + d0) = yu;
        *reinterpret_cast<V*>(y + d1) = yv;
    }
}

template <int DT, int VEC>
static void rope_launch(const RopeArgs& a, bool inter, hipStream_t st) {
    // four tokens a workgroup share the sincos phase's latency; short calls take one, for more workgroups
    const bool wide = a.T >= 2048;
    const dim3 grid(wide ? (a.T + 3) / 4 : a.T), block(kRopeThreads);
    if (wide && inter) hipLaunchKernelGGL((k_rope<DT, VEC, true, 4>), grid, block, 0, st, a);
    else if (wide) hipLaunchKernelGGL((k_rope<DT, VEC, false, 4>), grid, block, 0, st, a);
    else if (inter) hipLaunchKernelGGL((k_rope<DT, VEC, true, 1>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_rope<DT, VEC, false, 1>), grid, block, 0, st, a);
}

}  // namespace wf

using namespace wf;

extern "C" {

int wf_rotary_embed(const void* q, int64_t q_st, int64_t q_sh, int Hq, const void* k, int64_t k_st, int64_t k_sh, int Hk, int dtype,
                    const void* positions, int positions64, const double* freqs, int T, int D, int rotary_dim, int interleaved,
                    float scale, void* q_out, int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, void* stream) {
    WF_REQUIRE(dtype == WF_F32 || dtype == WF_BF16 || dtype == WF_F16, "rotary_embed: bad dtype %d", dtype);
    WF_REQUIRE(T >= 0 && Hq >= 0 && Hk >= 0, "rotary_embed: negative size (T %d, heads %d / %d)", T, Hq, Hk);
    WF_REQUIRE(T <= kMaxWgs256 && Hq <= 65535 && Hk <= 65535, "rotary_embed: too many tokens or heads (T %d, heads %d / %d)", T, Hq, Hk);
    WF_REQUIRE(D > 0 && D <= kRopeMaxDim, "rotary_embed: head_dim %d not in [1, %d]", D, kRopeMaxDim);
    WF_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= D, "rotary_embed: rotary_dim %d must be even, in [2, %d]",
               rotary_dim, D);
    if (T == 0 || Hq + Hk == 0) return WF_OK;
    WF_REQUIRE(positions && freqs && (Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)), "rotary_embed: null pointer");
    RopeArgs a{{q, k}, {q_out, k_out}, {q_st, k_st}, {q_sh, k_sh}, {qo_st, ko_st}, {qo_sh, ko_sh}, {Hq, Hk}, positions, positions64,
               freqs, T, D, rotary_dim, scale};
    const int vec = dtype == WF_F32 ? 4 : 8;
    bool wide = rotary_dim % (2 * vec) == 0 && D % vec == 0;
    for (int w = 0; w < 2; ++w)
        if (a.H[w])
            wide = wide && aligned16(a.x[w]) && aligned16(a.y[w]) && a.xt[w] % vec == 0 && a.xh[w] % vec == 0 && a.yt[w] % vec == 0 &&
                   a.yh[w] % vec == 0;
    hipStream_t st = as_stream(stream);
    if (dtype == WF_F32) wide ? rope_launch<DT_F32, 4>(a, interleaved, st) : rope_launch<DT_F32, 1>(a, interleaved, st);
    else if (dtype == WF_BF16) wide ? rope_launch<DT_BF16, 8>(a, interleaved, st) : rope_launch<DT_BF16, 1>(a, interleaved, st);
    else wide ? rope_launch<DT_F16, 8>(a, interleaved, st) : rope_launch<DT_F16, 1>(a, interleaved, st);
    return check_launch("rotary_embed");
}

}  // extern "C"
