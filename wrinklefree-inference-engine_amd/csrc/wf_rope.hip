// wf_rope.hip -- rotary positions on rows of q and k.
//
// Pair j of a head's first r dims, j < r / 2, is turned by the angle a = pos * freq[j]:
//     y1 = s (x1 cos a - x2 sin a),  y2 = s (x2 cos a + x1 sin a),
// pairs (j, j + r/2) (half layout) or (2j, 2j + 1) (interleaved), s one factor for all; dims >= r pass.
// The angle: positions reach millions of radians, where 32 bits have lost the fraction of a turn, so
// turns = pos * freq / 2pi are formed in 64 bits, the whole turns dropped there, and only the remainder
// in [-1/2, 1/2] goes to 32 bits (2^-25 of a half turn) and to sincospif. x is widened to 32 bits and each
// result rounded once. (cos and sin in 32 bits: f32 results are off by 3.9e-8 of their size (root mean square), 3.4e-8 where they are
// taken in 64; no difference in 16 bits.) A call reads and writes every element once and is bound by that.
//
// A workgroup takes four tokens (one in short calls): its threads first put the tokens' cos and sin
// in LDS, one sincos per (token, pair) for all heads, then walk the heads with two 16-byte loads and
// stores an item, whatever the strides, alignment and r; what r and D leave over goes one by one.
// Measured: 16384 tokens, 20 + 5 heads of 128, bf16: 45 us, 4.65 TB/s (a large copy: 4.90); 128 tokens 3.7 us on the
// device, latencies; 4097 tokens, 8 + 2 heads of 96, f32, interleaved 9.4 us; 10746
// tokens, 16 heads of 128 of which 58 turn, bf16: 33 us (76 element by element), of 80 with 40: 19 us (50).
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

// 16 bytes of a head, aligned as its elements are (global memory takes such accesses)
template <class T>
struct RopeVec {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(v, p, 16); }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, v, 16); }
};

template <int DT, bool INTER, int TOK>
__global__ __launch_bounds__(kRopeThreads) void k_rope(RopeArgs a) {
    using E = RopeElem<DT>;
    using T = typename E::T;
    using V = RopeVec<T>;
    constexpr int N = V::N;
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
    auto turn = [](T x1, T x2, float2 k, T& y1, T& y2) {
        const float u = E::up(x1), v = E::up(x2);
        y1 = E::down(fmaf(u, k.x, -(v * k.y)));
        y2 = E::down(fmaf(v, k.x, u * k.y));
    };
    // items of a head: N pairs each, then N passing dims each, then what is left of both one by one
    const int pairs = half / N, wide = pairs + (a.D - a.r) / N, ends = wide + half % N, per = ends + (a.D - a.r) % N, HT = a.H[0] + a.H[1];
    for (int i = threadIdx.x; i < nt * HT * per; i += kRopeThreads) {
        const int c = i % per, th = i / per, t = th / HT;
        int h = th - t * HT;
        const int w = h >= a.H[0];
        if (w) h -= a.H[0];
        const T* x = (const T*)a.x[w] + (t0 + t) * a.xt[w] + h * a.xh[w];
        T* y = (T*)a.y[w] + (t0 + t) * a.yt[w] + h * a.yh[w];
        if (c < pairs) {
            // the item's two vectors: dims [d0, +N) and [d1, +N)
            const int d0 = INTER ? 2 * N * c : N * c, d1 = INTER ? d0 + N : d0 + half;
            V u, v, yu, yv;
            u.load(x + d0);
            v.load(x + d1);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float2 k = cs[t][N * c + e];
                if constexpr (INTER) {  // element 2 e of the 2 N in order
                    V &from = 2 * e < N ? u : v, &to = 2 * e < N ? yu : yv;
                    turn(from.v[2 * e % N], from.v[2 * e % N + 1], k, to.v[2 * e % N], to.v[2 * e % N + 1]);
                } else {
                    turn(u.v[e], v.v[e], k, yu.v[e], yv.v[e]);
                }
            }
            yu.store(y + d0);
            yv.store(y + d1);
        } else if (c < wide) {
            const int d = a.r + (c - pairs) * N;
            V u;
            u.load(x + d);
            u.store(y + d);
        } else if (c < ends) {
            const int j = pairs * N + c - wide, d0 = INTER ? 2 * j : j, d1 = INTER ? d0 + 1 : d0 + half;
            T y1, y2;
            turn(x[d0], x[d1], cs[t][j], y1, y2);
            y[d0] = y1;
            y[d1] = y2;
        } else {
            const int d = a.D - (per - c);
            y[d] = x[d];
        }
    }
}

template <int DT>
static void rope_launch(const RopeArgs& a, bool inter, hipStream_t st) {
    // four tokens a workgroup share the sincos phase's latency; short calls take one, for more workgroups
    const bool wide = a.T >= 2048;
    const dim3 grid(wide ? (a.T + 3) / 4 : a.T), block(kRopeThreads);
    if (wide && inter) hipLaunchKernelGGL((k_rope<DT, true, 4>), grid, block, 0, st, a);
    else if (wide) hipLaunchKernelGGL((k_rope<DT, false, 4>), grid, block, 0, st, a);
    else if (inter) hipLaunchKernelGGL((k_rope<DT, true, 1>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_rope<DT, false, 1>), grid, block, 0, st, a);
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
    hipStream_t st = as_stream(stream);
    if (dtype == WF_F32) rope_launch<DT_F32>(a, interleaved, st);
    else if (dtype == WF_BF16) rope_launch<DT_BF16>(a, interleaved, st);
    else rope_launch<DT_F16>(a, interleaved, st);
    return check_launch("rotary_embed");
}

}  // extern "C"
