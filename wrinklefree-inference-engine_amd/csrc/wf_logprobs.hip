// wf_logprobs.hip -- log probabilities of given tokens, entropy and the top alternatives from logits.
//
// Row x of V logits, m = max x, Z = sum exp(x - m):
//     log p_t = x_t - m - log Z,     H = log Z - sum (x - m) exp(x - m) / Z,
//     rank of t = 1 + #{j : x_j > x_t} + #{j < t : x_j = x_t},  top k by value, the lower index first.
// Each logit has to be read once (2 bytes bf16), some 10 VALU cycles a logit and SIMD: bound by memory for
// many rows, by latency for few. One wave takes a chunk of one row and never meets another wave: no LDS,
// no barrier, no atomics, so results do not depend on timing. Per lane it keeps a running max and sums in
// the log2 domain, y = (x - max) log2e, e = 2^y, sum e and sum y e, rescaled when the lane's max rises.
//
// The top k without a data-dependent buffer: the chunk is cut into groups of four neighbouring 16-byte
// vectors (the four lanes of a quad); each group's max comes from the softmax's own max and two DPP steps.
// The k first groups, by (max, lower group first), hold the chunk's k first elements: an element of a
// later group is preceded by the maxima of k groups, each greater, or equal and further left. The wave
// keeps the k best groups sorted across its lanes (insertion: ballot, popcount, one lane shift), and reads
// just those k groups again at the end for the elements themselves. k <= 64 is the wave's width.
// A second launch, a wave per row, joins the chunks' sums and sorted lists.
#include "wf_common.h"
#include "wf_device.h"

namespace wf {

constexpr int kLpMaxTop = 64;
constexpr int kLpUnroll = 4;        // 16-byte vectors a lane holds of a tile
constexpr int kLpMaxSplits = 64;    // chunks of a row: a lane each in the join
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LpPart {  // one chunk's sums (z = 0: it holds nothing but -inf)
    float m, z, t;  // sum 2^y, sum y 2^y with y = (x - m) log2e
    int rank;       // elements of the chunk that come before the row's token
};

// The wave's k best (value, index) so far, sorted across lanes: value descending, lower index first.
// Empty places hold (-inf, INT_MAX), behind every real entry; a NaN never enters.
struct LpList {
    float v;
    int i;
    __device__ __forceinline__ LpList() : v(-INFINITY), i(0x7fffffff) {}
    static __device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }
    // the candidates (one a lane) that come before entry k - 1, one after the other
    __device__ __forceinline__ void add(float cv, int ci, int k) {
        float kv = __shfl(v, k - 1, 64);
        int ki = __shfl(i, k - 1, 64);
        for (uint64_t todo = __ballot(before(cv, ci, kv, ki)); todo;) {
            const int l = __builtin_ctzll(todo);
            const float nv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(cv), l));
            const int ni = __builtin_amdgcn_readlane(ci, l);
            const int at = __builtin_popcountll(__ballot(before(v, i, nv, ni))), lane = threadIdx.x & 63;
            const float pv = __shfl_up(v, 1, 64);
            const int pi = __shfl_up(i, 1, 64);
            v = lane < at ? v : lane == at ? nv : pv;
            i = lane < at ? i : lane == at ? ni : pi;
            kv = __shfl(v, k - 1, 64);
            ki = __shfl(i, k - 1, 64);
            todo &= todo - 1;
            todo &= __ballot(before(cv, ci, kv, ki));
        }
    }
};

template <int DT>
struct LpElem;  // logit type, logits of a 16-byte vector
template <>
struct LpElem<DT_F32> {
    using T = float;
    static constexpr int N = 4;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[N]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
};
template <>
struct LpElem<DT_BF16> {
    using T = uint16_t;
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(T v) { return bf2f(v); }
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[N]) {
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = bf_lo(d[e]), x[2 * e + 1] = bf_hi(d[e]);
    }
};
template <>
struct LpElem<DT_F16> {
    using T = uint16_t;
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(T v) { return h2f(v); }
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[N]) {
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = h2f(d[e] & 0xffffu), x[2 * e + 1] = h2f(d[e] >> 16);
    }
};

struct LpArgs {
    const void* x;
    int64_t ld;
    int R, V, S, chunk;  // chunks a row and logits a chunk
    const void* tok;
    int tok64, k;
    LpPart* part;   // [R][S]
    float* list_v;  // [R][S][k]
    int* list_i;
    float *lp, *ent, *top_v;
    int *rank, *top_i;
};

// The row's token, -1 when there is none to look for (no tokens asked, or outside [0, V)).
__device__ __forceinline__ int64_t lp_token(const LpArgs& a, int r) {
    if (!a.tok) return -1;
    return a.tok64 ? ((const int64_t*)a.tok)[r] : (int64_t)((const int32_t*)a.tok)[r];
}

// the next float above x: v >= above(x) exactly if v > x (NaN where nothing is above)
__device__ __forceinline__ float lp_above(float x) {
    if (!(x < INFINITY)) return NAN;
    x += 0.f;  // -0 -> +0
    const int b = __float_as_int(x);
    return __int_as_float(x >= 0.f ? b + 1 : b - 1);
}

// Running sums of one lane over the logits it has seen: z = sum 2^y, t = sum y 2^y, y = (x - m) log2e. The
// difference is taken before the product: m log2e overflows for logits at the type's lowest or highest value.
struct LpSums {
    float m, z, t;
    __device__ __forceinline__ LpSums() : m(-INFINITY), z(0.f), t(0.f) {}
    // x's frame: 0 while nothing but -inf (or NaN) was seen, so that -inf - m is no NaN
    __device__ __forceinline__ float frame() const { return m == -INFINITY ? 0.f : m; }
    // the sums in the frame of a max nm >= m; z = NaN stays
    __device__ __forceinline__ void move(float nm) {
        if (z == 0.f) return;
        const float d = (frame() - nm) * kLog2e, s = exp2f(d);
        t = s == 0.f ? 0.f : (t + d * z) * s;
        z *= s;
    }
    __device__ __forceinline__ void raise(float tm) {
        if (tm > m) {
            move(tm);
            m = tm;
        }
    }
    __device__ __forceinline__ void one(float x, float f) {
        const float y = (x - f) * kLog2e, e = __builtin_amdgcn_exp2f(y);
        z += e;
        t = fmaf(fmaxf(y, -200.f), e, t);  // y = -inf: 0, not NaN
    }
    // all lanes' sums in one frame (the max of those that hold something)
    __device__ __forceinline__ void join() {
        const float nm = wave_max(z == 0.f ? -INFINITY : m);
        move(nm == -INFINITY ? 0.f : nm);
        m = nm;
        z = wave_sum(z);
        t = wave_sum(t);
    }
};

template <int DT, bool TOP, bool TOK>
__global__ __launch_bounds__(256) void k_logprobs_part(LpArgs a) {
    using E = LpElem<DT>;
    constexpr int N = E::N, U = kLpUnroll;
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (w >= a.R * a.S) return;
    const int r = w / a.S, s = w - r * a.S;
    const typename E::T* row = (const typename E::T*)a.x + r * a.ld;
    const int lo = min(s * a.chunk, a.V), hi = min(lo + a.chunk, a.V);
    // whole 16-byte vectors of [lo, hi): [lo + head, lo + head + N nv); the rest (< 2 N logits) one a lane
    const int mis = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(typename E::T));
    const int head = min(mis ? N - mis : 0, hi - lo), nv = (hi - lo - head) / N, v0 = lo + head, tail = v0 + nv * N;
    int tok = -1;
    float xt = 0.f, gt = NAN;
    if constexpr (TOK) {
        const int64_t t = lp_token(a, r);
        tok = t >= 0 && t < a.V ? (int)t : -1;
        if (tok >= 0) {
            xt = E::up(row[tok]);
            gt = lp_above(xt);
        }
    }
    LpSums sum;
    LpList groups, elems;
    int rank = 0;  // of the wave, in a scalar
    // head and tail logits
    {
        const int j = lane < head ? lo + lane : lane < head + hi - tail ? tail + lane - head : -1;
        const float x = j >= 0 ? E::up(row[j]) : -INFINITY;
        sum.raise(x);
        if (j >= 0) sum.one(x, sum.frame());
        if constexpr (TOK) rank += __builtin_popcountll(__ballot(tok >= 0 && j >= 0 && (x > xt || (x == xt && j < tok))));
        if constexpr (TOP) elems.add(x, j >= 0 ? j : 0x7fffffff, a.k);
    }
    const uint4* vec = reinterpret_cast<const uint4*>(row + v0);
    uint4 nx[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u * 64 + lane < nv) nx[u] = vec[u * 64 + lane];
    for (int base = 0; base < nv; base += 64 * U) {
        uint4 cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u) cur[u] = nx[u];
#pragma unroll
        for (int u = 0; u < U; ++u) {  // the next tile's vectors are under way while this one is summed
            const int i = base + (U + u) * 64 + lane;
            if (i < nv) nx[u] = vec[i];
        }
        float x[U][N], vm[U], tm = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            E::unpack(cur[u], x[u]);
            const bool in = base + u * 64 + lane < nv;
#pragma unroll
            for (int e = 0; e < N; ++e) x[u][e] = in ? x[u][e] : -INFINITY;
            vm[u] = x[u][0];
#pragma unroll
            for (int e = 1; e < N; ++e) vm[u] = fmaxf(vm[u], x[u][e]);
            tm = fmaxf(tm, vm[u]);
        }
        sum.raise(tm);
        const float f = sum.frame();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) sum.one(x[u][e], f);
        if constexpr (TOK) {
            // before the token >= counts, from it on >; the vector that holds it one by one
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = base + u * 64 + lane, j = v0 + i * N;
                const bool hold = j <= tok && tok < j + N;
                const float lim = i >= nv || tok < 0 ? NAN : j + N <= tok ? xt : gt;
#pragma unroll
                for (int e = 0; e < N; ++e) rank += __builtin_popcountll(__ballot(x[u][e] >= lim));
                if (__ballot(hold && i < nv)) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        rank += __builtin_popcountll(__ballot(hold && i < nv && x[u][e] == xt && j + e < tok));
                }
            }
        }
        if constexpr (TOP) {
            // lane 4 g + u of a quad takes group g of vectors [64 u, 64 u + 64)
            float gm = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float m = fmaxf(vm[u], dpp_f<DPP_QP_1032>(vm[u]));
                m = fmaxf(m, dpp_f<DPP_QP_2301>(m));
                if ((lane & 3) == u) gm = m;
            }
            const int g = (base >> 2) + (lane & 3) * 16 + (lane >> 2);
            groups.add(gm, 4 * g < nv ? g : 0x7fffffff, a.k);
        }
    }
    sum.join();
    const int64_t at = (int64_t)r * a.S + s;
    if (lane == 0) a.part[at] = LpPart{sum.m, sum.z, sum.t, rank};
    if constexpr (TOP) {
        // the elements of the k best groups, 64 / (4 N) groups a round
        constexpr int G = 64 / (4 * N);
        for (int i = 0; i < a.k; i += G) {
            const int g = __shfl(groups.i, i + lane / (4 * N), 64);
            const int j = g == 0x7fffffff || i + lane / (4 * N) >= a.k ? hi : v0 + g * 4 * N + lane % (4 * N);
            const bool in = j < tail;
            if (!__ballot(in)) break;  // groups are sorted: none behind an empty place
            elems.add(in ? E::up(row[j]) : -INFINITY, in ? j : 0x7fffffff, a.k);
        }
        if (lane < a.k) {
            a.list_v[at * a.k + lane] = elems.v;
            a.list_i[at * a.k + lane] = elems.i;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_logprobs_join(LpArgs a) {
    using E = LpElem<DT>;
    const int r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (r >= a.R) return;
    const int64_t at = (int64_t)r * a.S;
    LpPart p{-INFINITY, 0.f, 0.f, 0};
    if (lane < a.S) p = a.part[at + lane];
    LpSums sum;
    sum.m = p.m, sum.z = p.z, sum.t = p.t;
    sum.join();
    const int rank = wave_sum_i(p.rank);
    const float lz = log2f(sum.z), ln_z = lz * kLn2;
    const bool empty = sum.z == 0.f;  // every logit is -inf
    if (lane == 0) {
        if (a.ent) a.ent[r] = empty ? 0.f : (lz - sum.t / sum.z) * kLn2;
        if (a.tok) {
            const int64_t tok = lp_token(a, r);
            const bool in = tok >= 0 && tok < a.V;
            const float x = in ? E::up(((const typename E::T*)a.x)[r * a.ld + tok]) : 0.f;
            a.lp[r] = tok < 0 ? 0.f : !in ? NAN : empty ? -INFINITY : x - sum.m - ln_z;
            a.rank[r] = in ? rank + 1 : 0;
        }
    }
    if (a.k == 0) return;
    // the chunks' sorted lists, a lane each, from the front until no front can enter
    LpList top;
    for (int i = 0; i < a.k; ++i) {
        float v = -INFINITY;
        int j = 0x7fffffff;
        if (lane < a.S) v = a.list_v[(at + lane) * a.k + i], j = a.list_i[(at + lane) * a.k + i];
        if (!__ballot(LpList::before(v, j, __shfl(top.v, a.k - 1, 64), __shfl(top.i, a.k - 1, 64)))) break;
        top.add(v, j, a.k);
    }
    if (lane < a.k) {
        const bool in = top.i != 0x7fffffff;  // no: fewer than k logits of the row are numbers
        a.top_i[(int64_t)r * a.k + lane] = in ? top.i : -1;
        a.top_v[(int64_t)r * a.k + lane] = !in ? NAN : empty ? -INFINITY : top.v - sum.m - ln_z;
    }
}

// Chunks a row: enough waves to fill the device (about 4096), but no chunk under a tile of a wave.
static int lp_splits(int R, int V) {
    const int64_t want = (4096 + (int64_t)R - 1) / R, most = ((int64_t)V + 2047) / 2048;
    return (int)max((int64_t)1, min(min(want, most), (int64_t)kLpMaxSplits));
}

template <int DT>
static void lp_launch(const LpArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.R * a.S + 3) / 4)), block(256);
    if (a.k && a.tok) hipLaunchKernelGGL((k_logprobs_part<DT, true, true>), grid, block, 0, st, a);
    else if (a.k) hipLaunchKernelGGL((k_logprobs_part<DT, true, false>), grid, block, 0, st, a);
    else if (a.tok) hipLaunchKernelGGL((k_logprobs_part<DT, false, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_logprobs_part<DT, false, false>), grid, block, 0, st, a);
    hipLaunchKernelGGL((k_logprobs_join<DT>), dim3((a.R + 3) / 4), block, 0, st, a);
}

}  // namespace wf

using namespace wf;

extern "C" {

int64_t wf_token_logprobs_ws_bytes(int R, int V, int top_k) {
    if (R <= 0 || V <= 0 || top_k < 0) return 0;
    return (int64_t)R * lp_splits(R, V) * (int64_t)(sizeof(LpPart) + 8 * (int64_t)top_k);
}

int wf_token_logprobs(const void* logits, int dtype, int64_t ld, int R, int V, const void* tokens, int tokens64, int top_k,
                      float* logprobs, int32_t* ranks, float* entropy, int32_t* top_ids, float* top_logprobs, void* ws, void* stream) {
    WF_REQUIRE(dtype == WF_F32 || dtype == WF_BF16 || dtype == WF_F16, "token_logprobs: bad dtype %d", dtype);
    WF_REQUIRE(R >= 0 && V > 0 && V <= 1 << 30, "token_logprobs: bad shape [%d, %d]", R, V);
    WF_REQUIRE(top_k >= 0 && top_k <= kLpMaxTop && top_k <= V, "token_logprobs: top_k %d not in [0, min(%d, vocabulary)]", top_k,
               kLpMaxTop);
    WF_REQUIRE(R == 0 || R == 1 || ld >= V, "token_logprobs: rows of %d logits at stride %lld", V, (long long)ld);
    if (R == 0) return WF_OK;
    WF_REQUIRE(logits && ws && aligned16(ws), "token_logprobs: null logits, or a workspace that is null or not 16-byte aligned");
    WF_REQUIRE(!tokens || (logprobs && ranks), "token_logprobs: null logprobs / ranks");
    WF_REQUIRE(top_k == 0 || (top_ids && top_logprobs), "token_logprobs: null top_ids / top_logprobs");
    const int S = lp_splits(R, V);
    WF_REQUIRE((int64_t)R * S <= 0x7fffffff - 4, "token_logprobs: too many rows");
    const int chunk = (int)((((int64_t)V + S - 1) / S + 31) / 32 * 32);
    LpPart* part = reinterpret_cast<LpPart*>(ws);
    float* list_v = reinterpret_cast<float*>(part + (int64_t)R * S);
    int* list_i = reinterpret_cast<int*>(list_v + (int64_t)R * S * top_k);
    LpArgs a{logits, ld, R, V, S, chunk, tokens, tokens64, top_k, part, list_v, list_i, logprobs, entropy, top_logprobs, ranks, top_ids};
    hipStream_t st = as_stream(stream);
    if (dtype == WF_F32) lp_launch<DT_F32>(a, st);
    else if (dtype == WF_BF16) lp_launch<DT_BF16>(a, st);
    else lp_launch<DT_F16>(a, st);
    return check_launch("token_logprobs");
}

}  // extern "C"
