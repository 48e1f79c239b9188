// wf_prefix.hip -- attention of one query token per sequence over the paged K/V pool, for batches whose
// sequences share a prefix: the prefix's keys are read once for all of them.
//
// Sequence b has L keys. Keys j < P stand on the pages of another row of the page table (the prefix's owner), the
// others on its own:  o = sum_j p_j v_j / l,  p_j = exp(scale q.k_j - m),  l = sum_j p_j,  lse = m + log l.
// The softmax splits over any partition of the keys into records (m, l, unnormalised o) that a second launch joins.
//
//   prefix  keys [0, P) of neighbouring sequences with the same owner and P ("shared"): a workgroup takes up to 32 query
//           rows (sequence, head of the kv group) and a range of the keys; every wave takes every fourth 32-key tile for
//           ALL rows, so a K/V byte is loaded once per 32 rows, straight into registers.
//   suffix  the other keys of a sequence (all of them where it shares with no neighbour): one kv head and a range of the
//           keys a workgroup, the group's heads as the matrix's columns. Bound by HBM.
//   join    one wave a (sequence, head): its records, the division, the output type.
// Prefix and suffix are the two kinds of workgroup of one launch, the join is a second.
//
// Tiles: the pool's 32-key K / V layouts (wf_norm.h k_tile_off / v_tile_off) are the A operands of the matrix cores as they
// lie: S^T (keys x rows) = K Q^T, whose accumulator leaves a lane with groups of 8 neighbouring keys of one row -- the B
// operand of O^T (dims x rows) = V^T P^T. Probabilities never leave their lane; no LDS and no barrier until the
// waves' records meet.
// The running max is raised only when a tile passes it by 2^8 (its exchange between the four lanes of a row and
// the rescaling of o are rare then): p <= 2^8 is as exact in bf16 and 32 bits as p <= 1.
//
// What bounds it: the loads and the arithmetic of a prefix wave follow each other, and it is alone on its SIMD. Issuing the 16 KiB
// (bf16) of a tile for 32 rows takes it some 1250 cycles beside the CU's three others (52 of the L1's 64 bytes a cycle), scores,
// softmax and products 425 + 370 + 454: 2500 cycles a tile, 86 tiles a wave behind 32768 keys. (A second prefix workgroup a CU
// loads no faster and was slower, see the launch rule.) Suffixes run at HBM's rate beside them. Measured a call, 20 query and 5 kv heads, bf16, batch 128:
// 1024 shared keys and suffixes to 512 (88 MB) 30 us, 35 where the inputs come round too late for the 256 MB cache in front of
// memory; 32768 and suffixes to 1024 (253 MB) 101 us; no sharing, 1024 keys each (335 MB) 59 us, 5.6 TB/s.
//
// Operands and rounding: scores, max, sums and o in 32 bits. The matrices are bf16, and f16 where q is f16 and the pool holds
// one-byte codes (all of them f16 values). Where the pool is bf16, an f16 q enters as the exact sum of two bf16 terms;
// an f32 q as three. P is rounded once to the output's type where that is the matrices' (bf16 2^-8, f16 2^-11 a
// term at most, as much as the output's own rounding; f16 with the exponents 7 higher, so that only p < 2^-21 lose bits,
// 2^-32 at most); else it has as many terms as q. What the one rounding costs: outputs off by 0.0018 (500 shared keys) to 0.0023
// (32768) of their size (root mean square), 0.0017 of it the output's own rounding; f16 over int8 0.00028, 0.00021 of it the output's. Who wants
// P in 32 bits passes q in f32: three terms each, at the cost given in pf_plan.
#include "wf_common.h"
#include "wf_device.h"
#include "wf_kv.h"

namespace wf {

typedef float pf_f4 __attribute__((ext_vector_type(4)));

constexpr int kPfDim = 128, kPfPage = 32;
constexpr int kPfMaxRecords = 64;          // splits of each part: a lane each in the join, twice
constexpr int kPfMinTiles = 4;             // tiles of a prefix range: one a wave at least (12: 64 pairs behind 512 keys 37 us, 33 with 4)
constexpr int kPfMinSuffix = 8;            // of a suffix range: two a wave
constexpr float kPfLn2 = 0.69314718055994530942f;

struct PfArgs {
    const void* q;
    int64_t q_sb, q_sh;
    int qvec;  // q's rows are 16-byte aligned
    const uint8_t *K, *V;
    int64_t pgs, hs;  // bytes from page to page and from head to head
    int np;
    const int32_t* pt;
    int64_t pts;
    int cols;
    const int32_t *lens, *owners, *plens;
    int B, Hq, Hkv, G;
    float sc, neg;  // |scale| log2e, and the sign that went to q
    float vs;
    int NP, NS;     // splits of the prefix and of the suffix; records of a row: NP + NS
    float2* ml;     // [B * Hq][NP + NS]
    float* o;       // [B * Hq][NP + NS][128]
    void* out;
    int64_t o_sb, o_sh;
    float* lse;
};

// A sequence's partition: keys [0, P) on owner's pages, [P, L) on its own.
struct PfSeq {
    int L, P, owner;
    __device__ __forceinline__ bool same(const PfSeq& s) const { return P > 0 && P == s.P && owner == s.owner; }
};
__device__ __forceinline__ PfSeq pf_seq(const PfArgs& a, int b) {
    const bool in = b >= 0 && b < a.B;
    const int i = in ? b : 0;  // no branch around the loads: three sequences' lengths are fetched at once
    const int len = a.lens[i], owner = a.owners[i], plen = a.plens[i];
    PfSeq s;
    s.L = in ? min(max(len, 0), a.cols * kPfPage) : 0;
    s.owner = in ? owner : -1;
    s.P = owner >= 0 && owner < a.B ? min(max(plen, 0), s.L) : 0;
    return s;
}
// Whether b's prefix is read together with a neighbour's (both launches ask this).
__device__ __forceinline__ bool pf_shared(const PfArgs& a, int b, const PfSeq& s) {
    return s.same(pf_seq(a, b - 1)) || s.same(pf_seq(a, b + 1));
}
// tiles of one of `splits` ranges, and how many ranges hold something
__device__ __forceinline__ int pf_per(int tiles, int splits, int least) { return max((tiles + splits - 1) / splits, least); }
__device__ __forceinline__ int pf_tiles(int keys) { return (keys + kPfPage - 1) / kPfPage; }

// The matrices' elements for a pool and q, and how many of them make up a q (and a p)
template <int KVQ, int QDT>
struct PfType {
    static constexpr bool kHalf = QDT == DT_F16 && KVQ != 0;
    static constexpr int kTerms = QDT == DT_BF16 || kHalf ? 1 : QDT == DT_F16 ? 2 : 3;
    using E = typename std::conditional<kHalf, _Float16, __bf16>::type;
    typedef E V8 __attribute__((ext_vector_type(8)));
    // 8 elements of a tile's fragment
    static constexpr int kBytes = KVQ == 0 ? 2 : 1;
    using T = typename std::conditional<KVQ == 0, uint4, uint2>::type;
    static __device__ __forceinline__ uint4 wide(T t) {
        if constexpr (KVQ == 0) return t;
        else if constexpr (KVQ == 1) return kHalf ? fp8x8_to_f16(t) : fp8x8_to_bf16(t);
        else return kHalf ? i8x8_to_f16(t) : i8x8_to_bf16_sext(t);
    }
};

// W query rows: the q fragments, running max, sum and output of one wave. A K or V tile is 8 fragments
// of 8 elements a lane, and either way the accumulator of S^T leaves a lane with the keys that it needs in P^T:
//   W = 16 (16x16x32 products): lane (l = row, g = quarter); scores of keys 8 g + e, e = 0..7;
//   W = 32 (32x32x16, 1.7 times the rate: 32 cycles to 2 x 27 measured): lane (l = row, g = half); scores of
//          keys 16 j + 8 g + e, j = 0, 1 -- K's 32 rows are the two 16-row halves of the tile one after the other.
template <int W, int KVQ, int QDT>
struct PfState {
    using Type = PfType<KVQ, QDT>;
    using E = typename Type::E;
    using V8 = typename Type::V8;
    using T = typename Type::T;
    static constexpr int N = Type::kTerms;
    static constexpr int J = W / 16;            // groups of 8 keys a lane
    static constexpr int M = kPfDim / W;        // accumulators
    static constexpr int S = W == 16 ? 4 : 8;   // dim steps of a score
    static constexpr float kUp = Type::kHalf ? 7.f : 0.f;  // the exponents' frame lies this much below the max: p < 2^(8 + 7), and normal in f16 from 2^-21 on
    typedef float Acc __attribute__((ext_vector_type(W == 16 ? 4 : 16)));
    V8 q[N][S];
    Acc acc[M];
    float m, f, l;  // max (log2 domain), the frame of the exponents (m - kUp, or 0 while it is -inf), sum

    static __device__ __forceinline__ int row() { return threadIdx.x & (W - 1); }
    static __device__ __forceinline__ int group() { return (threadIdx.x & 63) / W; }
    // where fragment i of this lane lies in a tile: K's (score step or half), V's (accumulator and key group)
    static __device__ __forceinline__ int k_at(int i) {
        if constexpr (W == 16) return i * 512 + (threadIdx.x & 63) * 8;  // i = 4 half + step
        else return (row() >> 4) * 2048 + i * 256 + group() * 128 + (row() & 15) * 8;
    }
    static __device__ __forceinline__ int v_at(int i) {
        if constexpr (W == 16) return i * 512 + (threadIdx.x & 63) * 8;
        else return (i >> 1) * 1024 + (row() >> 4) * 512 + (i & 1) * 256 + group() * 128 + (row() & 15) * 8;  // i = 2 m + j
    }
    static __device__ __forceinline__ Acc mfma(V8 x, V8 y, Acc c) {
        if constexpr (W == 16 && Type::kHalf) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
        else if constexpr (W == 16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
        else if constexpr (Type::kHalf) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }

    __device__ __forceinline__ void clear() {
        m = -INFINITY, f = 0.f, l = 0.f;
#pragma unroll
        for (int n = 0; n < M; ++n) acc[n] = Acc{};
    }
    // this lane's row; fragment c: its dims 8 (64 / W c + g) ..; vec: the row is 16-byte aligned
    __device__ __forceinline__ void load_q(const uint8_t* row, float neg, bool vec) {
        constexpr int G = 64 / W, V = QDT == DT_F32 ? 2 : 1;
#pragma unroll
        for (int c = 0; c < S; ++c) {
            float x[8];
            if (vec) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const uint4 w = reinterpret_cast<const uint4*>(row)[(G * c + group()) * V + i];
                    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (QDT == DT_F32) x[4 * i + e] = __uint_as_float(d[e]);
                        else if constexpr (QDT == DT_BF16) x[2 * e] = bf_lo(d[e]), x[2 * e + 1] = bf_hi(d[e]);
                        else x[2 * e] = h2f(d[e] & 0xffffu), x[2 * e + 1] = h2f(d[e] >> 16);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = load_as_f32(row, 8 * (G * c + group()) + e, QDT);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= neg;
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    q[k][c][e] = (E)x[e];
                    if (k + 1 < N) x[e] -= (float)q[k][c][e];
                }
        }
    }
    using Scores = float[8 * J];
    using Probs = V8[N][J];
    // scores of a 32-key tile: s[8 j + e] for key 8 (64 / W j + g) + e
    __device__ __forceinline__ void scores(const T (&kf)[8], Scores& s) {
        Acc c[W == 16 ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (W == 16 ? 2 : 1); ++h) c[h] = Acc{};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int step = W == 16 ? i >> 1 : i, h = W == 16 ? i & 1 : 0;
            const V8 kb = __builtin_bit_cast(V8, Type::wide(kf[W == 16 ? 4 * h + step : i]));
#pragma unroll
            for (int k = N - 1; k >= 0; --k) c[h] = mfma(kb, q[k][step], c[h]);
        }
#pragma unroll
        for (int e = 0; e < 8 * J; ++e)
            s[e] = W == 16 ? c[(e >> 2) & (W == 16)][e & 3] : c[0][(8 * ((e >> 2) & 1) + 4 * (e >> 3) + (e & 3)) & (W / 2 - 1)];
    }
    static __device__ __forceinline__ int key(int j) { return 8 * (64 / W * j + group()); }
    // scores -> probabilities in the rows' frames; keys outside [lo, hi) of the tile are masked
    __device__ __forceinline__ void softmax(Scores& x, Probs& p, int lo, int hi, float sc) {
        if (!(lo <= 0 && hi >= kPfPage)) {
            asm volatile("");  // a branch, not selects on every tile
#pragma unroll
            for (int e = 0; e < 8 * J; ++e) x[e] = key(e >> 3) + (e & 7) >= lo && key(e >> 3) + (e & 7) < hi ? x[e] : -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 8 * J; ++e) mx = fmaxf(mx, x[e]);
        mx *= sc;
        if (__any(mx > m + 8.f)) {
            if constexpr (W == 16) mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32, 64)), m);
            const float nf = mx == -INFINITY ? 0.f : mx - kUp;
            // (an empty sum stays, also when it is NaN: it holds no finite score to rescale)
            const float r = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(f - nf);
            l *= r;
#pragma unroll
            for (int n = 0; n < M; ++n) acc[n] *= r;
            m = mx;
            f = nf;
        }
#pragma unroll
        for (int e = 0; e < 8 * J; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], sc, -f));
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float* y = x + 8 * j;
            l += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < 8 * J; ++e) {
                p[k][e >> 3][e & 7] = (E)x[e];
                if (k + 1 < N) x[e] -= (float)p[k][e >> 3][e & 7];
            }
    }
    // o += P V
    __device__ __forceinline__ void values(const T (&vf)[8], const Probs& p, int lo, int hi) {
        uint4 v[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) v[n] = Type::wide(vf[n]);
        if (!(lo <= 0 && hi >= kPfPage)) {  // a masked key's V may hold anything: 0 x NaN is NaN
            asm volatile("");
#pragma unroll
            for (int j = 0; j < J; ++j) {
                uint32_t mask[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k0 = key(j) + 2 * i;
                    mask[i] = (k0 >= lo && k0 < hi ? 0xffffu : 0u) | (k0 + 1 >= lo && k0 + 1 < hi ? 0xffff0000u : 0u);
                }
#pragma unroll
                for (int n = j; n < 8; n += J) v[n] = make_uint4(v[n].x & mask[0], v[n].y & mask[1], v[n].z & mask[2], v[n].w & mask[3]);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const V8 vb = __builtin_bit_cast(V8, v[n]);
#pragma unroll
            for (int k = N - 1; k >= 0; --k) acc[n / J] = mfma(vb, p[k][n % J], acc[n / J]);
        }
    }
};

// One wave's walk over tiles k0, k0 + 4, .. below k1: page(k) is the page of tile k (per lane, k may differ by lane),
// range(k, lo, hi) its valid keys. 64 page ids are fetched at a time, a lane each. The next tile's K is under way from
// the moment this one's scores are done, its V from the moment this one's products are: one set of registers,
// and half a tile's work over each load's latency.
template <class State, class Page, class Range>
__device__ __forceinline__ void pf_walk(const PfArgs& a, State& st, const uint8_t* q, int64_t head, int k0, int k1, Page page, Range range) {
    using T = typename State::T;
    const int lane = threadIdx.x & 63, n = (k1 - k0 + 3) / 4;
    if (n <= 0) return;
    T kf[8], vf[8];
    int ids = k0 + 4 * lane < k1 ? page(k0 + 4 * lane) : -1;
    st.load_q(q, a.neg, a.qvec);  // beside the ids' latency, not before it
    ids = ids < a.np ? ids : -1;
    // the id of tile number i (0, 1, ..) of the walk; < 0 where the pool has no such page
    auto find = [&](int i) {
        if (i > 0 && (i & 63) == 0) {
            const int k = k0 + 4 * (i + lane);
            ids = k < k1 ? page(k) : -1;
            ids = ids < a.np ? ids : -1;
        }
        return __builtin_amdgcn_readlane(ids, i & 63);
    };
    auto load = [&](int id, const uint8_t* pool, T (&f)[8], bool v) {
        const uint8_t* p = pool + max(id, 0) * a.pgs + head;  // no such page: page 0, masked
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = *reinterpret_cast<const T*>(p + (v ? State::v_at(e) : State::k_at(e)) * State::Type::kBytes);
    };
    int id = find(0);
    load(id, a.K, kf, false);
    load(id, a.V, vf, true);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        int lo, hi;
        range(k0 + 4 * i, lo, hi);
        if (id < 0) hi = 0;
        id = i + 1 < n ? find(i + 1) : -1;
        typename State::Scores s;
        typename State::Probs p;
        st.scores(kf, s);
        load(id, a.K, kf, false);
        st.softmax(s, p, lo, hi, a.sc);
        st.values(vf, p, lo, hi);
        load(id, a.V, vf, true);
    }
}

// The four waves' states -> one record a row.
constexpr int kPfRow = kPfDim + 4;
template <int W>
struct __attribute__((aligned(16))) PfShared {
    float o[4][W][kPfRow];
    float m[4][W], l[4][W];
};
// row(i): the record's place in ml / o for row i of the wave's, or < 0; m: the frame of l and o, -inf where no score was finite
template <int W, class Acc, int M, class Row>
__device__ __forceinline__ void pf_merge(const PfArgs& a, PfShared<W>& sm, const Acc (&acc)[M], float m, float l, Row row) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & (W - 1), g = lane / W;
    if constexpr (W == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __syncthreads();  // the last run's records have been read
    // accumulator n, registers 4 i ..: dims W n + 8 i + 4 g .. (W = 16: i = 0)
#pragma unroll
    for (int n = 0; n < M; ++n)
#pragma unroll
        for (int i = 0; i < (W == 16 ? 1 : 4); ++i)
            *reinterpret_cast<pf_f4*>(&sm.o[wave][r][W * n + 8 * i + 4 * g]) = pf_f4{acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]};
    if (g == 0) sm.m[wave][r] = m, sm.l[wave][r] = l;
    __syncthreads();
    // 256 / W threads a row, 8 dims each at a time
    constexpr int T = 256 / W;
    const int y = threadIdx.x / T;
    const int64_t rec = row(y);
    if (rec < 0) return;
    float mm = -INFINITY, w[4], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) mm = fmaxf(mm, sm.m[i][y]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // a wave that saw no finite score has l = 0 (or NaN) in the frame 0
        w[i] = mm == -INFINITY ? 1.f : sm.m[i][y] == -INFINITY ? (sm.l[i][y] == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(sm.m[i][y] - mm);
        sum += sm.l[i][y] * w[i];
    }
#pragma unroll
    for (int d = (threadIdx.x % T) * 4; d < kPfDim; d += 4 * T) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += sm.o[i][y][d + e] * w[i];
        *reinterpret_cast<float4*>(a.o + rec * kPfDim + d) = make_float4(x[0], x[1], x[2], x[3]);
    }
    if (threadIdx.x % T == 0) a.ml[rec] = make_float2(mm, sum);
}

// ---------------------------------------------------------------------------------------------
// Shared prefixes. A workgroup per (kv head, key range, tile of MT rows) and turn. A tile's rows are taken in runs of
// sequences with one prefix, in 16 or 32 rows.
// ---------------------------------------------------------------------------------------------
template <int KVQ, int QDT, int W>
__device__ __forceinline__ void pf_run(const PfArgs& a, void* lds, int h, int z, int64_t ra, int64_t rb, int P, int owner, int k0, int k1) {
    PfState<W, KVQ, QDT> st;
    const int64_t r = min(ra + st.row(), rb - 1);
    const int b = (int)(r / a.G), g = (int)(r - (int64_t)b * a.G);
    const uint8_t* q = (const uint8_t*)a.q + (b * a.q_sb + (int64_t)(h * a.G + g) * a.q_sh) * (QDT == DT_F32 ? 4 : 2);
    st.clear();
    const int32_t* row = a.pt + owner * a.pts;
    pf_walk(a, st, q, h * a.hs, k0 + (int)(threadIdx.x >> 6), k1, [&](int k) { return row[k]; },
            [&](int k, int& lo, int& hi) { lo = 0, hi = P - k * kPfPage; });
    pf_merge(a, *static_cast<PfShared<W>*>(lds), st.acc, st.m - st.kUp, st.l, [&](int i) -> int64_t {
        if (ra + i >= rb) return -1;
        const int64_t b = (ra + i) / a.G;
        return (b * a.Hq + h * a.G + (ra + i - b * a.G)) * (a.NP + a.NS) + z;
    });
}

template <int KVQ, int QDT, int MT>
__device__ void pf_prefix(const PfArgs& a, void* lds, int h, int z, int tile, int turn, int turns) {  // runs turn, turn + turns, .. of the tile
    const int lane = threadIdx.x & 63;
    const int64_t r0 = (int64_t)tile * MT, r1 = min(r0 + MT, (int64_t)a.B * a.G);
    const int b0 = (int)(r0 / a.G), b1 = (int)((r1 - 1) / a.G);  // sequences of the tile: at most MT <= 32
    // lane i: sequence b0 + i
    const int bl = b0 + lane <= b1 ? b0 + lane : -2;
    const PfSeq me = pf_seq(a, bl), before = pf_seq(a, bl - 1), after = pf_seq(a, bl + 1);
    uint64_t todo = __ballot(me.same(before) || me.same(after));
    const uint64_t joined = __ballot(me.same(before));
    while (todo) {
        // a run of neighbours with one prefix: sequences b0 + i .. b0 + j - 1
        const int i = __builtin_ctzll(todo);
        const uint64_t stop = i == 63 ? ~0ull : ~(joined >> (i + 1));
        const int j = min(i + 1 + (int)__builtin_ctzll(stop | 1ull << 63), b1 - b0 + 1);
        todo &= j >= 64 ? 0ull : ~0ull << j;
        const int P = __builtin_amdgcn_readlane(me.P, i), owner = __builtin_amdgcn_readlane(me.owner, i);
        const int tiles = pf_tiles(P), per = pf_per(tiles, a.NP, kPfMinTiles);
        const int k0 = z * per, k1 = min(k0 + per, tiles);
        if (turn != 0) {  // another workgroup's run
            --turn;
            continue;
        }
        turn = turns - 1;
        if (k0 >= k1) continue;  // the whole workgroup
        const int64_t ra = max(r0, (int64_t)(b0 + i) * a.G), rb = min(r1, (int64_t)(b0 + j) * a.G);  // its rows
        if constexpr (MT > 16)
            if (rb - ra > 16) {
                pf_run<KVQ, QDT, 32>(a, lds, h, z, ra, rb, P, owner, k0, k1);
                continue;
            }
        pf_run<KVQ, QDT, 16>(a, lds, h, z, ra, rb, P, owner, k0, k1);
    }
}

// ---------------------------------------------------------------------------------------------
// The other keys. Block (key range z, kv head and tile of 16 of its heads, sequence).
// ---------------------------------------------------------------------------------------------
template <int KVQ, int QDT>
__device__ void pf_suffix(const PfArgs& a, void* lds, int z, int hc, int b) {
    const int ct = hc / a.Hkv, h = hc - ct * a.Hkv;
    const PfSeq s = pf_seq(a, b);
    // tiles [0, n1) the owner's, below P; then its own from the tile that holds P on
    const int n1 = pf_shared(a, b, s) ? 0 : pf_tiles(s.P), first = s.P / kPfPage;
    const int tiles = s.L > s.P ? n1 + pf_tiles(s.L) - first : n1;
    const int per = pf_per(tiles, a.NS, kPfMinSuffix), k0 = z * per, k1 = min(k0 + per, tiles);
    if (k0 >= k1) return;
    PfState<16, KVQ, QDT> st;
    const int g = min(ct * 16 + st.row(), a.G - 1);
    const uint8_t* q = (const uint8_t*)a.q + (b * a.q_sb + (int64_t)(h * a.G + g) * a.q_sh) * (QDT == DT_F32 ? 4 : 2);
    st.clear();
    pf_walk(a, st, q, h * a.hs, k0 + (int)(threadIdx.x >> 6), k1,
            [&](int k) { return a.pt[(k < n1 ? s.owner : b) * a.pts + (k < n1 ? k : first + k - n1)]; },
            [&](int k, int& lo, int& hi) {
                const int at = (k < n1 ? k : first + k - n1) * kPfPage;
                lo = k < n1 ? 0 : s.P - at;
                hi = (k < n1 ? s.P : s.L) - at;
            });
    pf_merge(a, *static_cast<PfShared<16>*>(lds), st.acc, st.m - st.kUp, st.l, [&](int i16) -> int64_t {
        const int g = ct * 16 + i16;
        return g < a.G ? ((int64_t)b * a.Hq + h * a.G + g) * (a.NP + a.NS) + a.NP + z : -1;
    });
}

// The first np workgroups the prefixes, in row tiles of MT; the others the other keys: the one part waits for the
// matrix cores and L1, the other for HBM.
template <int KVQ, int QDT, int MT>
__global__ __launch_bounds__(256, 2) void k_shared_prefix(PfArgs a, int np, int turns) {
    __shared__ PfShared<MT> sm;
    int x = blockIdx.x;
    if (x < np) {
        // consecutive workgroups go round the 8 XCDs: each takes an eighth of the list (head, range, row tile, turn), so that
        // the row tiles of one (head, range) meet in one L2, or in two neighbours' (whole groups to an XCD: 160 sequences
        // of 20 query and 5 kv heads behind 32768 keys 152 us, 115 so)
        const int tiles = (int)(((int64_t)a.B * a.G + MT - 1) / MT), i = (x & 7) * (np >> 3) + (x >> 3);
        const int u = i / turns, g = u / tiles, h = g / a.NP;
        if (h < a.Hkv) pf_prefix<KVQ, QDT, MT>(a, &sm, h, g - h * a.NP, u - g * tiles, i - u * turns, turns);
        return;
    }
    x -= np;
    const int hc = a.Hkv * ((a.G + 15) / 16), z = x % a.NS, y = x / a.NS;
    pf_suffix<KVQ, QDT>(a, &sm, z, y % hc, y / hc);
}

// ---------------------------------------------------------------------------------------------
// The join: a wave per (sequence, head), lane i the dims 2 i, 2 i + 1.
// ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_prefix_join(PfArgs a, int odt) {
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= (int64_t)a.B * a.Hq) return;
    const int b = (int)(row / a.Hq), hq = (int)(row - (int64_t)b * a.Hq);
    // Records of a row stand at fixed places, NP of the prefix's ranges and NS of the suffix's: their sums and the first records
    // are under way before the lengths say which of them were written.
    const int R = a.NP + a.NS;
    const float2* ml = a.ml + row * R;
    const float2* o = reinterpret_cast<const float2*>(a.o + row * R * kPfDim) + lane;
    const float2 none = make_float2(-INFINITY, 0.f);
    float2 e0 = lane < R ? ml[lane] : none, e1 = lane + 64 < R ? ml[lane + 64] : none;
    const float2 o_prefix = o[0], o_suffix = o[a.NP * (kPfDim / 2)];
    const PfSeq s = pf_seq(a, b);
    const bool sh = pf_shared(a, b, s);
    const int tp = sh ? pf_tiles(s.P) : 0, pp = pf_per(tp, a.NP, kPfMinTiles), np = (tp + pp - 1) / pp;
    const int n1 = sh ? 0 : pf_tiles(s.P), ts = s.L > s.P ? n1 + pf_tiles(s.L) - s.P / kPfPage : n1;
    const int ps = pf_per(ts, a.NS, kPfMinSuffix), ns = (ts + ps - 1) / ps;
    auto written = [&](int i) { return i < a.NP ? i < np : i - a.NP < ns; };
    e0 = written(lane) ? e0 : none;
    e1 = written(lane + 64) ? e1 : none;
    const float M = wave_max(fmaxf(e0.x, e1.x));
    auto weight = [&](float2 e) {
        return M == -INFINITY ? 1.f : e.x == -INFINITY ? (e.y == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(e.x - M);
    };
    const float w0 = weight(e0), w1 = weight(e1), L = wave_sum(e0.y * w0 + e1.y * w1);
    float x = 0.f, y = 0.f;
    auto add = [&](int i, float2 v) {
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(i < 64 ? w0 : w1), i & 63));
        x += v.x * w;
        y += v.y * w;
    };
    auto part = [&](int first, int n, float2 v0) {
        if (n > 0) add(first, v0);
        for (int i = 1; i < n; i += 4) {
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) v[k] = o[(first + i + k) * (kPfDim / 2)];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) add(first + i + k, v[k]);
        }
    };
    part(0, np, o_prefix);
    part(a.NP, ns, o_suffix);
    // no key, or none with a score above -inf: zeros
    const float inv = L == 0.f ? 0.f : a.vs / L;
    const int64_t at = b * a.o_sb + hq * a.o_sh + 2 * lane;
    store_from_f32(a.out, at, odt, L == 0.f ? 0.f : x * inv);
    store_from_f32(a.out, at + 1, odt, L == 0.f ? 0.f : y * inv);
    if (a.lse && lane == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kPfLn2;
}

struct PfPlan {
    int MT, NP, NS;  // rows of a prefix workgroup, splits
    int turns;       // workgroups of a row tile and range, which take its runs in turn
    int64_t np, ns;  // workgroups
};
// Launch shape from what the host knows: whether q is one term (at most as many ranges where it is not), rows, kv heads and the table's width (an upper bound of every length).
static PfPlan pf_plan(bool one, int B, int Hq, int Hkv, int cols) {
    const int64_t rows = (int64_t)B * (Hq / Hkv), groups = (Hq / Hkv + 15) / 16;
    PfPlan p;
    // 32 rows of a q of several terms would leave one workgroup a CU its registers: 4096 shared keys 48 us (f32) and 42 (f16), 36 and
    // 33 with 16 rows (a smaller batch), short prefixes 33 -> 23. 128 sequences of 20 and 5 heads over a bf16 pool, behind 4096 keys / 32768: 41 us /
    // 101 in bf16, 46 / 231 in f16, 47 / 234 in f32 (half the rows a load serves, two and three times the products)
    p.MT = rows <= 16 || !one ? 16 : 32;
    const int64_t tiles = (rows + p.MT - 1) / p.MT;
    auto clamp = [](int64_t v, int64_t hi) { return (int)max((int64_t)1, min(min(v, hi), (int64_t)kPfMaxRecords)); };
    // prefix ranges: one workgroup a CU. A second one reads no faster (L1: 52 bytes a cycle with one), and its place goes to a suffix
    // workgroup, whose time is HBM's: 32768 shared keys 102 us, 118 with two.
    p.NP = clamp(256 / (tiles * Hkv), (cols + kPfMinTiles - 1) / kPfMinTiles);
    p.NS = clamp(512 / ((int64_t)B * Hkv * groups), (cols + 1 + kPfMinSuffix - 1) / kPfMinSuffix);
    // runs of a tile on workgroups of their own while there are CUs for them: 30 sequences in 4 groups 27 -> 16 us, 19 in 8 20 -> 16
    const int64_t w = (int64_t)Hkv * p.NP * tiles;
    p.turns = (int)max((int64_t)1, min(256 / w, (int64_t)min(B / 2, 8)));
    p.np = B > 1 ? (w * p.turns + 7) / 8 * 8 : 0;  // one sequence shares nothing
    p.ns = p.NS * Hkv * groups * B;
    return p;
}

template <int KVQ, int QDT>
static void pf_launch(const PfArgs& a, const PfPlan& p, int odt, hipStream_t st) {
    const dim3 grid((unsigned)(p.np + p.ns)), block(256);
    constexpr int kWide = PfType<KVQ, QDT>::kTerms == 1 ? 32 : 16;
    if (p.MT == 16) hipLaunchKernelGGL((k_shared_prefix<KVQ, QDT, 16>), grid, block, 0, st, a, (int)p.np, p.turns);
    else hipLaunchKernelGGL((k_shared_prefix<KVQ, QDT, kWide>), grid, block, 0, st, a, (int)p.np, p.turns);
    hipLaunchKernelGGL(k_prefix_join, dim3((unsigned)(((int64_t)a.B * a.Hq + 3) / 4)), block, 0, st, a, odt);
}

template <int KVQ>
static void pf_dispatch(const PfArgs& a, const PfPlan& p, int dt, hipStream_t st) {
    if (dt == DT_BF16) pf_launch<KVQ, DT_BF16>(a, p, dt, st);
    else if (dt == DT_F16) pf_launch<KVQ, DT_F16>(a, p, dt, st);
    else pf_launch<KVQ, DT_F32>(a, p, dt, st);
}

}  // namespace wf

using namespace wf;

extern "C" {

int64_t wf_shared_prefix_attention_ws_bytes(int dtype, int B, int Hq, int Hkv, int max_blocks) {
    if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_blocks <= 0) return 0;
    const PfPlan p = pf_plan(dtype != WF_F32, B, Hq, Hkv, max_blocks);  // f16: one term over some pools
    return (int64_t)B * Hq * (p.NP + p.NS) * (int64_t)(sizeof(float2) + 4 * kPfDim);
}

int wf_shared_prefix_attention(const void* q, int dtype, int64_t q_sb, int64_t q_sh, const void* k_pool, const void* v_pool, int kv_quant,
                               int64_t page_stride, int64_t head_stride, int num_pages, const int32_t* page_table,
                               int64_t table_stride, int max_blocks, const int32_t* seq_lens, const int32_t* prefix_rows,
                               const int32_t* prefix_lens, float k_scale, float v_scale, float sm_scale, int B, int Hq, int Hkv, int D,
                               void* out, int64_t o_sb, int64_t o_sh, float* lse, void* ws, void* stream) {
    WF_REQUIRE(dtype == WF_F32 || dtype == WF_BF16 || dtype == WF_F16, "shared_prefix_attention: bad dtype %d", dtype);
    WF_REQUIRE(kv_quant == WF_KV_BF16 || kv_quant == WF_KV_FP8 || kv_quant == WF_KV_INT8, "shared_prefix_attention: bad kv_quant %d", kv_quant);
    WF_REQUIRE(D == kPfDim, "shared_prefix_attention: the pool's tile layouts need head_dim 128 (got %d)", D);
    WF_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "shared_prefix_attention: bad heads or batch (B %d, Hq %d, Hkv %d)", B, Hq, Hkv);
    WF_REQUIRE(B <= 65535 && (int64_t)Hkv * ((Hq / Hkv + 15) / 16) <= 65535 && (int64_t)B * (Hq / Hkv) <= 16 * 65535,
               "shared_prefix_attention: batch %d or heads %d / %d too many", B, Hq, Hkv);
    WF_REQUIRE(num_pages > 0 && max_blocks > 0 && max_blocks <= 0x7fffffff / kPfPage && table_stride >= max_blocks,
               "shared_prefix_attention: bad pool or table (%d pages, rows of %d at stride %lld)", num_pages, max_blocks, (long long)table_stride);
    const int eb = kv_quant == WF_KV_BF16 ? 2 : 1;
    WF_REQUIRE(page_stride >= 0 && head_stride >= 0 && page_stride * eb % 16 == 0 && head_stride * eb % 16 == 0,
               "shared_prefix_attention: page and head strides must be multiples of 16 bytes");
    const float sc = sm_scale * k_scale * 1.44269504088896340736f;
    WF_REQUIRE(fabsf(sc) > 0.f && fabsf(sc) < INFINITY, "shared_prefix_attention: sm_scale %g times k_scale %g must be finite, not 0", sm_scale,
               k_scale);
    if (B == 0) return WF_OK;
    WF_REQUIRE(q && k_pool && v_pool && page_table && seq_lens && prefix_rows && prefix_lens && out && ws,
               "shared_prefix_attention: null pointer");
    WF_REQUIRE(aligned16(k_pool) && aligned16(v_pool) && aligned16(ws), "shared_prefix_attention: pools and workspace must be 16-byte aligned");
    const PfPlan p = pf_plan(dtype == WF_BF16 || (dtype == WF_F16 && kv_quant != WF_KV_BF16), B, Hq, Hkv, max_blocks);
    WF_REQUIRE(p.np + p.ns <= kMaxWgs256 && (int64_t)B * Hq <= 4 * kMaxWgs256, "shared_prefix_attention: batch %d with heads %d / %d too many", B, Hq,
               Hkv);
    const int64_t recs = (int64_t)B * Hq * (p.NP + p.NS);
    float* o = reinterpret_cast<float*>(ws);
    const int per16 = dtype == WF_F32 ? 4 : 8;
    PfArgs a{q, q_sb, q_sh, aligned16(q) && q_sb % per16 == 0 && q_sh % per16 == 0, (const uint8_t*)k_pool, (const uint8_t*)v_pool, page_stride * eb, head_stride * eb, num_pages, page_table,
             table_stride, max_blocks, seq_lens, prefix_rows, prefix_lens, B, Hq, Hkv, Hq / Hkv, fabsf(sc), sc < 0.f ? -1.f : 1.f, v_scale,
             p.NP, p.NS, reinterpret_cast<float2*>(o + recs * kPfDim), o, out, o_sb, o_sh, lse};
    hipStream_t st = as_stream(stream);
    if (kv_quant == WF_KV_BF16) pf_dispatch<0>(a, p, dtype, st);
    else if (kv_quant == WF_KV_FP8) pf_dispatch<1>(a, p, dtype, st);
    else pf_dispatch<2>(a, p, dtype, st);
    return check_launch("shared_prefix_attention");
}

}  // extern "C"
