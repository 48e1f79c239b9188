// wf_logprobs.hip -- log probabilities of given tokens, entropy and the top alternatives from logits.
//
// Row x of V logits, m = max x, Z = sum exp(x - m):
//     log p_t = x_t - m - log Z,     H = log Z - sum (x - m) exp(x - m) / Z,
//     rank of t = 1 + #{j : x_j > x_t} + #{j < t : x_j = x_t},  top k by value, the lower index first.
// Each logit has to be read once (2 bytes bf16), some 14 VALU cycles a logit and SIMD: bound by memory for
// many rows, by latency for few. One wave takes a chunk of one row and never meets another wave: no
// barrier, no atomics, so results do not depend on timing. Per lane it keeps a running max and sums in
// the log2 domain, y = (x - max) log2e, e = 2^y, sum e and sum y e, rescaled when the lane's max rises.
// A second launch, a wave per row, joins the chunks' sums and sorted lists.
//
// The top k without a data-dependent buffer, from maxima that the sums need anyway:
//   short chunks (4096 logits, few rows) stay in registers. The k-th greatest of the 64 lanes' maxima bounds the k-th
//     logit from below; what reaches it (some 64 ln(64 / (64 - k)) logits; from k = 33 on the vectors'
//     maxima are taken instead) is packed by ballots and ordered once.
//   long chunks are cut into groups of four neighbouring 16-byte vectors (the four lanes of a quad), each group's max two
//     DPP steps more. The k first groups, by (max, lower group first), hold the chunk's k first elements: an
//     element of a later group is preceded by the maxima of k groups, each greater, or equal and further left. The
//     wave keeps the k best groups sorted across its lanes and reads just those again at the end. k <= 64 is the wave's width.
// Rounding: 32 bits throughout, a lane's sums one logit after the other (up to a thousand for a prompt's rows) with the hardware's
// exp2: log probabilities of 2048 rows are off by 1.3e-7 of their size (root mean square), where whole rows summed as a tree are off by 5e-8.
// Measured, vocabulary 128256 in bf16: 2048 rows with 5 alternatives 117 us, 4.5 TB/s (109 us, 4.8 TB/s, without any); 128 rows
// with 20: 17 us and 5 of the join (the reading and summing alone 11.7); one row 6.6 + 3.8 us, latencies.
#include "wf_common.h"
#include "wf_device.h"

namespace wf {

constexpr int kLpMaxTop = 64;
constexpr int kLpUnroll = 4;        // 16-byte vectors a lane holds of a tile
constexpr int kLpHeld = 4096;       // logits of a chunk that stay in registers: 2 tiles of 16 bits, 4 of 32
constexpr int kLpPlaces = 128;      // places for what may be among their alternatives
constexpr int kLpMergeLists = 16;   // chunks of a row up to which the join merges whole lists
constexpr int kLpMaxSplits = 64;    // chunks of a row: a lane each in the join
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LpPart {  // one chunk's sums (z = 0: it holds nothing but -inf)
    float m, z, t;  // sum 2^y, sum y 2^y with y = (x - m) log2e
    int rank;       // elements of the chunk that come before the row's token
};

// lane ^ X of a wave: DPP within 16 lanes, an LDS permute beyond
template <int X>
__device__ __forceinline__ int lp_xor(int v) {
    if constexpr (X == 1) return dpp_i<DPP_QP_1032>(v);
    else if constexpr (X == 2) return dpp_i<DPP_QP_2301>(v);
    else if constexpr (X == 3) return dpp_i<0x1B>(v);  // quad_perm 3, 2, 1, 0
    else if constexpr (X == 4) return dpp_i<DPP_HALF_MIRROR>(dpp_i<0x1B>(v));
    else if constexpr (X == 7) return dpp_i<DPP_HALF_MIRROR>(v);
    else if constexpr (X == 8) return dpp_i<DPP_ROW_ROR8>(v);
    else if constexpr (X == 15) return dpp_i<DPP_MIRROR>(v);
    else return __shfl_xor(v, X, 64);
}
template <int X>
__device__ __forceinline__ double lp_xor(double v) {
    return __hiloint2double(lp_xor<X>(__double2hiint(v)), lp_xor<X>(__double2loint(v)));
}
constexpr int kDppWaveShr1 = 0x138;  // lane l reads lane l - 1

// A logit and its index as one key that orders them (value descending, lower index first, +0 = -0), so that a step of a sort
// is one max and one min: 32 bits in the values' order above 2^31 - 1 - index, read as a double. From -inf to
// +inf these are positive normal doubles (exponents 3 to 0x7fc); 0 stands for no entry, and for NaN.
__device__ __forceinline__ double lp_key(float v, int i) {
    const uint32_t b = __float_as_uint(v + 0.f), o = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
    return v == v ? __longlong_as_double((long long)((uint64_t)o << 31 | (uint32_t)(0x7fffffff - i))) : 0.;
}
__device__ __forceinline__ float lp_value(double k) {
    const uint32_t o = (uint32_t)((uint64_t)__double_as_longlong(k) >> 31);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int lp_index(double k) { return 0x7fffffff - (int)(__double2loint(k) & 0x7fffffff); }

// The wave's greatest keys so far, descending across its lanes.
struct LpList {
    double v;
    __device__ __forceinline__ LpList() : v(0.) {}
    // one step of a bitonic network: of lanes l and l ^ X, the one without bit BIT keeps the greater key
    template <int X, int BIT>
    static __device__ __forceinline__ void step(double& v) {
        const double w = lp_xor<X>(v), hi = __builtin_fmax(v, w), lo = __builtin_fmin(v, w);
        v = threadIdx.x & BIT ? lo : hi;
    }
    template <int X>
    static __device__ __forceinline__ void clean(double& v) {
        step<X, X>(v);
        if constexpr (X > 1) clean<X / 2>(v);
    }
    static __device__ __forceinline__ void sort(double& v) {
        step<1, 1>(v);
        step<3, 2>(v), clean<1>(v);
        step<7, 4>(v), clean<2>(v);
        step<15, 8>(v), clean<4>(v);
        step<31, 16>(v), clean<8>(v);
        step<63, 32>(v), clean<16>(v);
    }
    // with another sorted list
    __device__ __forceinline__ void merge(double c) {
        v = __builtin_fmax(v, lp_xor<63>(c));  // the first 64 of both, a bitonic sequence
        clean<32>(v);
    }
    static __device__ __forceinline__ double lane(double v, int l) {
        return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
    }
    __device__ __forceinline__ double last(int k) const { return lane(v, k - 1); }  // entry k - 1
    // Takes in the candidates (one a lane) above entry k - 1: many by a sort and a merge (27 steps of the network), few one
    // after the other.
    __device__ __forceinline__ void add(double c, int k) {
        uint64_t todo = __ballot(c > last(k));
        if (__builtin_popcountll(todo) > 8) {
            c = todo >> (threadIdx.x & 63) & 1 ? c : 0.;
            sort(c);
            merge(c);
            return;
        }
        while (todo) {
            const double n = lane(c, __builtin_ctzll(todo));
            const int at = __builtin_popcountll(__ballot(v > n)), l = threadIdx.x & 63;
            const double p = __hiloint2double(dpp_i<kDppWaveShr1>(__double2hiint(v)), dpp_i<kDppWaveShr1>(__double2loint(v)));
            v = l < at ? v : l == at ? n : p;
            todo &= todo - 1;
            todo &= __ballot(c > last(k));
        }
    }
};

// LDS of one wave: its accesses are in order, the compiler's too
__device__ __forceinline__ void lp_meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// The first 64 of the n <= P keys in the wave's P places (P = 64, 128), a lane each: a key's place is the number of greater ones.
template <int P>
__device__ __forceinline__ double lp_order(double* q, int n) {
    const int lane = threadIdx.x & 63;
    lp_meet();
    double c[P / 64];
    int at[P / 64], keys = 0;  // keys: without those of no entry
#pragma unroll
    for (int h = 0; h < P / 64; ++h) {
        c[h] = lane + 64 * h < n ? q[lane + 64 * h] : 0.;
        at[h] = 0;
        keys += __builtin_popcountll(__ballot(c[h] > 0.));
    }
    lp_meet();
#pragma unroll
    for (int h = 0; h < P / 64; ++h) q[lane + 64 * h] = c[h];
    lp_meet();
#pragma unroll 1
    for (int i = 0; i < n; i += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double k = q[i + e];
#pragma unroll
            for (int h = 0; h < P / 64; ++h) at[h] += k > c[h];
        }
    lp_meet();
#pragma unroll
    for (int h = 0; h < P / 64; ++h)
        if (c[h] > 0. && at[h] < 64) q[at[h]] = c[h];
    lp_meet();
    const double v = lane < keys ? q[lane] : 0.;
    lp_meet();
    return v;
}

// Candidates on their way to a list: packed into the wave's 64 places in LDS by a ballot and a lane count each, taken in
// together when the places are full or at the end.
struct LpQueue {
    double* q;
    int n;  // of the wave, in a scalar
    __device__ __forceinline__ explicit LpQueue(double* places) : q(places), n(0) {}
    __device__ __forceinline__ void flush(LpList& l, int k) {
        if (!(l.last(1) > 0.)) {
            l.v = lp_order<64>(q, n);
            n = 0;
            return;
        }
        lp_meet();
        const double c = (int)(threadIdx.x & 63) < n ? q[threadIdx.x & 63] : 0.;
        lp_meet();
        n = 0;
        l.add(c, k);
    }
    // the place of this lane's key among those of `in`
    __device__ __forceinline__ int place(uint64_t in) const {
        return n + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
    }
    // the lanes' keys where `in`
    __device__ __forceinline__ void push(uint64_t in, double c, LpList& l, int k) {
        if (n + __builtin_popcountll(in) > 64) flush(l, k);
        if (in >> (threadIdx.x & 63) & 1) q[place(in)] = c;
        n += __builtin_popcountll(in);
    }
};

// dword i of a lane's vectors (registers: a tree of selects)
template <int U>
__device__ __forceinline__ uint32_t lp_dword(const uint4 (&w)[U], int i) {
    uint32_t d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t lo = i & 1 ? w[u].y : w[u].x, hi = i & 1 ? w[u].w : w[u].z;
        d[u] = i & 2 ? hi : lo;
    }
#pragma unroll
    for (int n = U, b = 4; n > 1; n /= 2, b *= 2)
#pragma unroll
        for (int u = 0; u < n / 2; ++u) d[u] = i & b ? d[2 * u + 1] : d[2 * u];
    return d[0];
}

template <int DT>
struct LpElem;  // logit type, logits of a 16-byte vector
template <>
struct LpElem<DT_F32> {
    using T = float;
    static constexpr int N = 4;
    static __device__ __forceinline__ float up(T v) { return v; }
    static __device__ __forceinline__ uint32_t bits(T v) { return __float_as_uint(v); }
    // the vector's first logit; the vector without it
    static __device__ __forceinline__ float pop(uint4& w) {
        const float x = __uint_as_float(w.x);
        w = make_uint4(w.y, w.z, w.w, 0);
        return x;
    }
    // logit p of the lane's U vectors
    template <int U>
    static __device__ __forceinline__ float pick(const uint4 (&w)[U], int p) { return __uint_as_float(lp_dword(w, p)); }
    static __device__ __forceinline__ void unpack(uint4 w, float (&x)[N]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
};
template <>
struct LpElem<DT_BF16> {
    using T = uint16_t;
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(T v) { return bf2f(v); }
    static __device__ __forceinline__ uint32_t bits(T v) { return v; }
    static __device__ __forceinline__ float pop(uint4& w) {
        const float x = bf2f(w.x & 0xffffu);
        w = make_uint4(__builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16), __builtin_amdgcn_alignbit(w.w, w.z, 16),
                       w.w >> 16);
        return x;
    }
    // logit p of the lane's U vectors
    template <int U>
    static __device__ __forceinline__ float pick(const uint4 (&w)[U], int p) {
        const uint32_t d = lp_dword(w, p >> 1);
        return p & 1 ? bf_hi(d) : bf_lo(d);
    }
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
    static __device__ __forceinline__ uint32_t bits(T v) { return v; }
    static __device__ __forceinline__ float pop(uint4& w) {
        const float x = h2f(w.x & 0xffffu);
        w = make_uint4(__builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16), __builtin_amdgcn_alignbit(w.w, w.z, 16),
                       w.w >> 16);
        return x;
    }
    // logit p of the lane's U vectors
    template <int U>
    static __device__ __forceinline__ float pick(const uint4 (&w)[U], int p) {
        const uint32_t d = lp_dword(w, p >> 1);
        return h2f(p & 1 ? d >> 16 : d & 0xffffu);
    }
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
    double* list;   // [R][S][k] keys
    float *lp, *ent, *top_v;
    int *rank, *top_i;
};

// The row's token, -1 when there is none to look for (no tokens asked, or outside [0, V)).
__device__ __forceinline__ int64_t lp_token(const LpArgs& a, int r) {
    if (!a.tok) return -1;
    typedef const __attribute__((address_space(4))) int32_t* P;  // constant while the kernel runs: a scalar load
    const P p = (P)(uintptr_t)a.tok;
    return a.tok64 ? (int64_t)((uint64_t)(uint32_t)p[2 * (int64_t)r + 1] << 32 | (uint32_t)p[2 * (int64_t)r]) : (int64_t)p[r];
}

// the next float above x: v >= above(x) exactly if v > x (NaN where nothing is above)
__device__ __forceinline__ float lp_above(float x) {
    if (!(x < INFINITY)) return NAN;
    x += 0.f;  // -0 -> +0
    const int b = __float_as_int(x);
    return __int_as_float(x >= 0.f ? b + 1 : b - 1);
}

// Running sums of one lane over the logits it has seen: z = sum 2^y, t = sum y 2^y, y = (x - m) log2e + c. In the
// loop y is one fma, x log2e - g with g = m log2e rounded; c = m log2e - g is what the rounding took and goes back in when
// the frame moves. Where m log2e might overflow (logits near the type's lowest or highest value) c is 0 and the
// difference is taken first.
struct LpSums {
    float m, c, z, t;
    __device__ __forceinline__ LpSums() : m(-INFINITY), c(0.f), z(0.f), t(0.f) {}
    // 0 while nothing but -inf (or NaN) was seen, so that -inf - m is no NaN
    __device__ __forceinline__ float frame() const { return m == -INFINITY ? 0.f : m; }
    static __device__ __forceinline__ bool huge(float f) { return !(fabsf(f) < 1e30f); }
    // the sums in the frame (nm, nc), nm >= m; z = NaN stays
    __device__ __forceinline__ void move(float nm, float nc) {
        if (z != 0.f) {
            const float d = (frame() - nm) * kLog2e - c + nc, s = exp2f(d);
            t = s == 0.f ? 0.f : (t + d * z) * s;
            z *= s;
        }
        c = nc;
    }
    __device__ __forceinline__ void raise(float tm) {
        if (tm > m) {
            move(tm, huge(tm) ? 0.f : fmaf(tm, kLog2e, -(tm * kLog2e)));
            m = tm;
        }
    }
    __device__ __forceinline__ void sum(float y) {
        const float e = __builtin_amdgcn_exp2f(y);
        z += e;
        t = fmaf(fmaxf(y, -200.f), e, t);  // y = -inf: 0, not NaN (a NaN stays in z)
    }
    // N logits whose max is not above m (the caller raised it)
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N]) {
        const float f = frame();
        if (__ballot(huge(f))) {
#pragma unroll
            for (int e = 0; e < N; ++e) sum(fmaf(x[e] - f, kLog2e, c));
        } else {
            const float g = f * kLog2e;
#pragma unroll
            for (int e = 0; e < N; ++e) sum(fmaf(x[e], kLog2e, -g));
        }
    }
    // all lanes' sums in one frame (the max of those that hold something)
    __device__ __forceinline__ void join() {
        const float nm = wave_max(z == 0.f ? -INFINITY : m);
        move(nm == -INFINITY ? 0.f : nm, 0.f);
        m = nm;
        z = wave_sum(z);
        t = wave_sum(t);
    }
};

// At most the k-th greatest of the lanes' M values each (no NaN), to 16 bits of it
template <int M>
__device__ __forceinline__ float lp_kth(const float (&v)[M], int k) {
    uint32_t o[M], at = 0;
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const uint32_t b = __float_as_uint(v[m]);
        o[m] = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);  // in the values' order
    }
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int m = 0; m < M; ++m) n += __builtin_popcountll(__ballot(o[m] >= (at | bit)));
        if (n >= k) at |= bit;
    }
    at = max(at, 0x007fffffu);  // -inf
    return __uint_as_float(at & 0x80000000u ? at ^ 0x80000000u : ~at);
}

// HELD (TOP): the chunk has at most kLpHeld logits, which stay in registers.
template <int DT, bool TOP, bool TOK, bool HELD>
__global__ __launch_bounds__(256) void k_logprobs_part(LpArgs a) {
    using E = LpElem<DT>;
    constexpr int N = E::N, U = kLpUnroll;
    __shared__ double places[4][HELD ? kLpPlaces : 64];
    const int w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (w >= a.R * a.S) return;
    const int r = w / a.S, s = w - r * a.S;
    const typename E::T* row = (const typename E::T*)a.x + r * a.ld;
    const int lo = min(s * a.chunk, a.V), hi = min(lo + a.chunk, a.V);
    // whole 16-byte vectors of [lo, hi): [lo + head, lo + head + N nv); the rest (< 2 N logits) one a lane
    const int mis = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(typename E::T));
    const int head = min(mis ? N - mis : 0, hi - lo), nv = (hi - lo - head) / N, v0 = lo + head, tail = v0 + nv * N;
    LpSums sum;
    LpQueue queue(places[threadIdx.x >> 6]);
    int rank = 0;  // of the wave, in a scalar
    const uint4* vec = reinterpret_cast<const uint4*>(row + v0);
    auto load = [&](int base, uint4 (&to)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (base + u * 64 + lane < nv) to[u] = ldg_nt(reinterpret_cast<const uint8_t*>(vec + base + u * 64 + lane));
    };
    // Loads return in order: the first tile, the token's logit, what is left of the chunk, so that nothing waits for more than
    // it needs. The token itself comes through the scalar cache.
    constexpr int H = HELD ? kLpHeld / (64 * U * N) : 1;
    uint4 held[H][U];
    load(0, held[0]);
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
    // head and tail logits
    const int edge = lane < head ? lo + lane : lane < head + hi - tail ? tail + lane - head : -1;
    typename E::T edge_x = 0;
    if (edge >= 0) edge_x = row[edge];
#pragma unroll
    for (int t = 1; t < H; ++t) load(64 * U * t, held[t]);
    // a tile's logits, -inf behind the chunk's last
    auto unpack = [&](int base, const uint4 (&from)[U], float (&x)[U][N]) {
        const bool whole = base + 64 * U <= nv;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            E::unpack(from[u], x[u]);
            if (!whole) {
                const bool in = base + u * 64 + lane < nv;
#pragma unroll
                for (int e = 0; e < N; ++e) x[u][e] = in ? x[u][e] : -INFINITY;
            }
        }
    };
    // the sums and the rank over a tile; vm: its vectors' maxima
    auto take = [&](int base, const float (&x)[U][N], float (&vm)[U]) {
        float tm = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vm[u] = x[u][0];
#pragma unroll
            for (int e = 1; e < N; ++e) vm[u] = fmaxf(vm[u], x[u][e]);
            tm = fmaxf(tm, vm[u]);
        }
        sum.raise(tm);
#pragma unroll
        for (int u = 0; u < U; ++u) sum.add(x[u]);
        if constexpr (TOK) {
            // before the token >= counts, from it on >; the vector that holds it one by one
            if (tok >= 0 && __any(tm >= xt)) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = base + u * 64 + lane, j = v0 + i * N;
                    const bool hold = j <= tok && tok < j + N && i < nv;
                    const float lim = i >= nv ? NAN : j + N <= tok ? xt : gt;
#pragma unroll
                    for (int e = 0; e < N; ++e) rank += __builtin_popcountll(__ballot(x[u][e] >= lim));
                    if (__any(hold)) {
#pragma unroll
                        for (int e = 0; e < N; ++e) rank += __builtin_popcountll(__ballot(hold && x[u][e] == xt && j + e < tok));
                    }
                }
            }
        }
        return tm;
    };
    const int64_t at = (int64_t)r * a.S + s;
    if constexpr (HELD) {
        float x[U][N], vm[H * U], most[1] = {-INFINITY};
#pragma unroll
        for (int v = 0; v < H * U; ++v) vm[v] = -INFINITY;
#pragma unroll
        for (int t = 0; t < H; ++t) {
            if (64 * U * t >= nv) break;
            unpack(64 * U * t, held[t], x);
            float tv[U];
            most[0] = fmaxf(most[0], take(64 * U * t, x, tv));
#pragma unroll
            for (int u = 0; u < U; ++u) vm[U * t + u] = fmaxf(-INFINITY, tv[u]);
        }
        // k lanes' maxima reach the k-th of them: nothing below it is among the k first. What reaches it is packed into the
        // queue's places: some 64 ln(64 / (64 - k)) logits; beyond k = 32, of the vectors' maxima, little more than k.
        float least = a.k <= 32 ? lp_kth(most, a.k) : lp_kth(vm, a.k);
        // for the signs below: -0 - 0 has one, and both zeros reach 0; less -0 neither has. inf - inf is a NaN with a sign of its own;
        // inf less the greatest number is not, and what else that lets in the keys leave behind
        if (least == 0.f) least = -0.f;
        least = fminf(least, 0x1.fffffep127f);
        if (least == -INFINITY) queue.n = kLpPlaces + 1;  // also logits of -inf, whose difference has no sign
        LpList elems;
        auto pack = [&](bool in, float v, int j) {
            const uint64_t go = __ballot(in);
            if (go) {
                const int to = queue.place(go);
                if (in && to < kLpPlaces) queue.q[to] = lp_key(v, j);
                queue.n += __builtin_popcountll(go);
            }
        };
        {
            const float v = edge >= 0 ? E::up(edge_x) : 0.f;
            pack(edge >= 0 && v >= least, v, edge);
        }
#pragma unroll
        for (int t = 0; t < H; ++t) {
            if (64 * U * t >= nv || queue.n > kLpPlaces) break;
            unpack(64 * U * t, held[t], x);
            // which of the lane's U N logits reach it, the first at the top: the differences' signs, two instructions a logit (a
            // NaN logit's sign may be either: its key is that of no entry)
            uint32_t mine = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) mine = __builtin_amdgcn_alignbit(mine, __float_as_uint(x[u][e] - least), 31);
            mine = ~mine << (32 - U * N);
            const int there = (nv - 64 * U * t - lane + 63) / 64 * N;  // the lane's logits up to the chunk's end
            if (there < U * N) mine &= there > 0 ? ~(0xffffffffu >> there) : 0u;
            while (queue.n <= kLpPlaces && __any(mine)) {
                const int p = __builtin_clz(mine | 1u), j = v0 + (64 * (U * t + p / N) + lane) * N + p % N;
                pack(mine != 0, E::pick(held[t], p), j);
                mine &= ~(0x80000000u >> p);
            }
        }
        if (queue.n <= kLpPlaces) {
            elems.v = queue.n > 64 ? lp_order<kLpPlaces>(queue.q, queue.n) : lp_order<64>(queue.q, queue.n);
        } else {  // many equal ones, or the greatest in few lanes: again, a full queue's at a time, from memory
            queue.n = 0;
            uint4 w = make_uint4(E::bits(edge_x), 0, 0, 0);
            int j = edge, n = 1;
#pragma unroll 1
            for (int b = 0;; b += 64) {
#pragma unroll 1
                for (int e = 0; e < n; ++e) {
                    const float v = E::pop(w);
                    const double c = lp_key(v, j + e);
                    const uint64_t in = __ballot(j >= 0 && v >= least && c > elems.last(a.k));
                    if (in) queue.push(in, c, elems, a.k);
                }
                if (b >= nv) break;
                n = N;
                j = b + lane < nv ? v0 + (b + lane) * N : -1;
                if (j >= 0) w = vec[b + lane];
            }
            queue.flush(elems, a.k);
        }
        if (lane < a.k) a.list[at * a.k + lane] = elems.v;
    } else {
        LpList groups;
        uint4 (&nx)[U] = held[0];
        for (int base = 0; base < nv; base += 64 * U) {
            uint4 cur[U];
#pragma unroll
            for (int u = 0; u < U; ++u) cur[u] = nx[u];
            load(base + 64 * U, nx);  // under way while this tile is summed
            float x[U][N], vm[U];
            unpack(base, cur, x);
            take(base, x, vm);
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
                const double c = 4 * g < nv ? lp_key(gm, g) : 0.;
                const uint64_t in = __ballot(c > groups.last(a.k));
                if (in) queue.push(in, c, groups, a.k);
            }
        }
        if constexpr (TOP) {
            // the k best groups again, a vector a lane, 16 groups a load, and before them the head and tail logits; one copy of
            // the list's code in a rolled loop: unrolled, fetching instructions took longer than running them
            queue.flush(groups, a.k);
            // k maxima reach the k-th: nothing below it is among the k first
            const double kth = groups.last(a.k);
            const float least = kth > 0. ? lp_value(kth) : -INFINITY;
            LpList elems;
            auto fetch = [&](int i, uint4& w, int& j) {
                const int e = 16 * i + (lane >> 2);
                const double c = __shfl(groups.v, e, 64);
                const int vi = 4 * lp_index(c) + (lane & 3);
                j = e < a.k && c > 0. && vi < nv ? v0 + vi * N : -1;
                if (j >= 0) w = vec[vi];
            };
            uint4 w = make_uint4(E::bits(edge_x), 0, 0, 0), w1 = w;
            int j = edge, n = 1, j1;
            fetch(0, w1, j1);
#pragma unroll 1
            for (int i = 1;; ++i) {
#pragma unroll 1
                for (int e = 0; e < n; ++e) {
                    const float x = E::pop(w);
                    const uint64_t in = __ballot(j >= 0 && x >= least);
                    if (in) queue.push(in, lp_key(x, j + e), elems, a.k);
                }
                if (16 * (i - 1) >= a.k) break;
                w = w1, j = j1, n = N;
                if (16 * i < a.k) fetch(i, w1, j1);
            }
            queue.flush(elems, a.k);
            if (lane < a.k) a.list[at * a.k + lane] = elems.v;
        }
    }
    {  // the head and tail logits
        const float x = edge >= 0 ? E::up(edge_x) : -INFINITY;
        sum.raise(x);
        const float one[1] = {x};
        sum.add(one);
        if constexpr (TOK) rank += __builtin_popcountll(__ballot(tok >= 0 && edge >= 0 && (x > xt || (x == xt && edge < tok))));
    }
    sum.join();
    if (lane == 0) a.part[at] = LpPart{sum.m, sum.z, sum.t, rank};
}

template <int DT>
__global__ __launch_bounds__(256) void k_logprobs_join(LpArgs a) {
    using E = LpElem<DT>;
    __shared__ double places[4][64];
    const int r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (r >= a.R) return;
    const int64_t at = (int64_t)r * a.S;
    LpPart p{-INFINITY, 0.f, 0.f, 0};
    if (lane < a.S) p = a.part[at + lane];
    // the chunks' sorted lists, a lane each
    const double* list = a.list + (at + lane) * a.k;
    auto fetch = [&](int i) { return lane < a.S && i < a.k ? list[i] : 0.; };
    double c0 = fetch(0), c1 = fetch(1), c2 = fetch(2);
    auto whole = [&](int i) { return lane < a.k && i < a.S ? a.list[(at + i) * a.k + lane] : 0.; };
    LpSums sum;
    sum.m = p.m, sum.z = p.z, sum.t = p.t;
    sum.join();
    const int rank = wave_sum_i(p.rank);
    const bool empty = sum.z == 0.f;  // every logit is -inf
    // the greatest logit's own term is 1: a sum that the frames' roundings left below would make a sure token's log probability positive
    if (sum.z < 1.f && !empty) sum.z = 1.f;
    const float lz = log2f(sum.z), ln_z = lz * kLn2, ent = (lz - sum.t / sum.z) * kLn2;
    if (lane == 0) {
        if (a.ent) a.ent[r] = empty || ent < 0.f ? 0.f : ent;
        if (a.tok) {
            const int64_t tok = lp_token(a, r);
            const bool in = tok >= 0 && tok < a.V;
            const float x = in ? E::up(((const typename E::T*)a.x)[r * a.ld + tok]) : 0.f;
            a.lp[r] = tok < 0 ? 0.f : !in ? NAN : empty ? -INFINITY : x - sum.m - ln_z;
            a.rank[r] = in ? rank + 1 : 0;
        }
    }
    if (a.k == 0) return;
    // The heads first: of what follows in the lists only what comes before the k-th so far can enter, from the fronts until
    // no front can.
    LpList top;
    LpQueue queue(places[threadIdx.x >> 6]);
    if (a.S > kLpMergeLists) {
        queue.push(__ballot(c0 > 0.), c0, top, a.k);
        queue.flush(top, a.k);
#pragma unroll 1
        for (int i = 1; i < a.k; ++i) {
            const uint64_t in = __ballot(c1 > top.last(a.k));
            if (!in) break;
            queue.push(in, c1, top, a.k);
            c1 = c2;
            c2 = fetch(i + 2);
        }
        queue.flush(top, a.k);
    } else {
        // few lists go deep: merged one after the other
        top.v = whole(0);
        double next = whole(1);
#pragma unroll 1
        for (int i = 1; i < a.S; ++i) {
            const double c = next;
            next = whole(i + 1);
            top.merge(c);
        }
    }
    if (lane < a.k) {
        const bool in = top.v > 0.;  // no: fewer than k logits of the row are numbers
        a.top_i[(int64_t)r * a.k + lane] = in ? lp_index(top.v) : -1;
        a.top_v[(int64_t)r * a.k + lane] = !in ? NAN : empty ? -INFINITY : lp_value(top.v) - sum.m - ln_z;
    }
}

// Chunks a row: as many waves as the device holds at once, 4096, or a few less (535 rows of 155893 with 20 alternatives: 7
// chunks 57 us, 8 leave a second round of 184 waves, 66); more where fewer would leave a seventh of it empty. More also where
// that makes the chunks short enough for registers, up to 6144 waves (404 rows of 55653 37 -> 30 us), or 12288 where there is
// a second round anyway. At most a chunk for every 2048 logits (V = 2049: two of them, half a tile of 16 bits each).
static int lp_splits(int R, int V) {
    const int64_t down = 4096 / (int64_t)R, fit = R * down >= 3500 ? down : (4096 + (int64_t)R - 1) / R;
    const int64_t held = ((int64_t)V + kLpHeld - 1) / kLpHeld, want = R * held <= (R * fit > 4096 ? 12288 : 6144) ? max(fit, held) : fit;
    return (int)max((int64_t)1, min(min(want, ((int64_t)V + 2047) / 2048), (int64_t)kLpMaxSplits));
}

template <int DT>
static void lp_launch(const LpArgs& a, bool held, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.R * a.S + 3) / 4)), block(256);
    if (a.k && a.tok && held) hipLaunchKernelGGL((k_logprobs_part<DT, true, true, true>), grid, block, 0, st, a);
    else if (a.k && held) hipLaunchKernelGGL((k_logprobs_part<DT, true, false, true>), grid, block, 0, st, a);
    else if (a.k && a.tok) hipLaunchKernelGGL((k_logprobs_part<DT, true, true, false>), grid, block, 0, st, a);
    else if (a.k) hipLaunchKernelGGL((k_logprobs_part<DT, true, false, false>), grid, block, 0, st, a);
    else if (a.tok) hipLaunchKernelGGL((k_logprobs_part<DT, false, true, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_logprobs_part<DT, false, false, false>), grid, block, 0, st, a);
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
    const int S = lp_splits(R, V), chunk = (int)((((int64_t)V + S - 1) / S + 31) / 32 * 32);
    const bool held = chunk <= kLpHeld;
    WF_REQUIRE((int64_t)R * S <= 4 * kMaxWgs256, "token_logprobs: too many rows (%d)", R);
    LpPart* part = reinterpret_cast<LpPart*>(ws);
    LpArgs a{logits, ld, R, V, S, chunk, tokens, tokens64, top_k, part, reinterpret_cast<double*>(part + (int64_t)R * S), logprobs, entropy, top_logprobs, ranks, top_ids};
    hipStream_t st = as_stream(stream);
    if (dtype == WF_F32) lp_launch<DT_F32>(a, held, st);
    else if (dtype == WF_BF16) lp_launch<DT_BF16>(a, held, st);
    else lp_launch<DT_F16>(a, held, st);
    return check_launch("token_logprobs");
}

}  // extern "C"
