// wf_plan.hip -- block tables and slot maps of a paged KV cache, built on the device from request lengths.
//
// Sequence b holds c tokens and gets n more, pages of p tokens: it has ceil(c / p) pages and needs
// ceil((c + n) / p) of them; the missing ones come from `free_pages` at the exclusive sum of what the
// sequences before it need. Token i of b stands at position c + i: entry (c + i) div p of its table row,
// slot (c + i) mod p. Everything is a prefix sum over B lengths and then 16 bytes of output per token, so
// a call is latency (one launch) up to some 100k tokens and the stores' bandwidth beyond.
//
// One launch: every workgroup repeats the prefix sum over all B lengths in LDS (8 bytes read per sequence,
// from L2) and then fills its own tokens and table rows; a separate scan launch would cost more than the
// repetition as long as the lengths fit LDS (kPlanLdsSeqs). Above that one workgroup scans into a workspace.
// Measured on the device: 128 sequences with one token each 3.9 us; 1024 sequences with 768k tokens 8.6 us, 12 MB of them
// stores (2.5 us at a copy's rate), the rest one chain of latencies: lengths, sums, search, page, store. 5000 sequences with 40k
// tokens 7.8 us of the scan and 11.5; 50000 with 400k 68.5 and 15: one workgroup scans, 1024 sequences in some 1.4 us.
#include "wf_common.h"
#include "wf_device.h"

namespace wf {

constexpr int kPlanThreads = 256;
constexpr int kPlanLdsSeqs = 2048;   // four int32 arrays of this many and one more in LDS (32 KiB)
constexpr int kPlanWide = 1 << 15;   // tokens from which a thread takes four neighbours (16-byte stores) instead of one

struct PlanArgs {
    const int32_t *cached, *fresh;
    int B;
    const int32_t* free_pages;
    int F;
    int32_t* table;
    int64_t ts;
    int cols, page, shift, T;  // shift: log2 of page, or -1
    int32_t *pages, *slots, *rows, *pos, *cu, *counts;
    int32_t *ws_off, *ws_cu;  // [B + 1] each, B > kPlanLdsSeqs only
    int lens16;               // both length arrays are 16-byte aligned
};

// Lengths are clamped to >= 0; sums are 64 bits and saturate where they are stored as 32.
__device__ __forceinline__ int32_t sat32(int64_t v) { return (int32_t)(v < 0x7fffffff ? v : 0x7fffffff); }
__device__ __forceinline__ uint32_t plan_div(const PlanArgs& a, uint32_t v) { return a.shift >= 0 ? v >> a.shift : v / (uint32_t)a.page; }

struct PlanSeq {
    uint32_t c, n;        // held and new tokens
    uint32_t have;        // pages held
    uint32_t need;        // pages missing, 0 if lng
    bool lng;             // does not fit the table row
    // pages [off, off + need) of the free list are there
    __device__ __forceinline__ bool fit(int64_t off, int F) const { return !lng && (need == 0 || off + need <= F); }
};
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int c, int n) {
    PlanSeq s;
    s.c = (uint32_t)max(c, 0);
    s.n = (uint32_t)max(n, 0);
    const uint32_t up = (uint32_t)a.page - 1;
    s.have = plan_div(a, s.c + up);                     // c + up < 2^32
    const uint32_t total = s.c + s.n;                   // < 2^32
    const uint32_t q = plan_div(a, total), blocks = q + (q * (uint32_t)a.page < total);
    s.lng = blocks > (uint32_t)a.cols;
    s.need = s.lng ? 0 : blocks - s.have;
    return s;
}

// inclusive sum over the wave's lanes (DPP: rows of 16, then across rows)
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t plan_add(int64_t v) {
    const uint32_t lo = (uint32_t)dpp_i<CTRL, ROWS>((int)(uint32_t)v, 0), hi = (uint32_t)dpp_i<CTRL, ROWS>((int)(v >> 32), 0);
    return v + (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t plan_wave_sum(int64_t v) {
    v = plan_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v = plan_add<0x112, 0xF>(v);
    v = plan_add<0x114, 0xF>(v);
    v = plan_add<0x118, 0xF>(v);
    v = plan_add<DPP_BCAST15, 0xA>(v);
    return plan_add<DPP_BCAST31, 0xC>(v);
}

// Exclusive sums of need and n over all sequences into off[0..B], cu[0..B], a thread taking E neighbours of every
// 256 E; lengths into cl, nl where a workgroup keeps them. `report`: this workgroup leaves the counts.
template <int E>
__device__ void plan_scan(const PlanArgs& a, int32_t* off, int32_t* cu, int32_t* cl, int32_t* nl, bool report) {
    __shared__ int64_t sm_n[4], sm_t[4];
    __shared__ int sh_taken, sh_refused;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) sh_taken = sh_refused = 0;
    int64_t cn = 0, ct = 0;  // sums before this round
    int taken = 0, refused = 0;
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads * E) {
        PlanSeq s[E];
        int64_t n = 0, t = 0;
        int c[E], f[E];
        const int bt = b0 + E * threadIdx.x;
        if (E == 4 && a.lens16 && bt + 4 <= a.B) {
            const int4 v = *reinterpret_cast<const int4*>(a.cached + bt), w = *reinterpret_cast<const int4*>(a.fresh + bt);
            c[0] = v.x, c[E / 4] = v.y, c[E / 2] = v.z, c[E - 1] = v.w;
            f[0] = w.x, f[E / 4] = w.y, f[E / 2] = w.z, f[E - 1] = w.w;
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                c[i] = bt + i < a.B ? a.cached[bt + i] : 0;
                f[i] = bt + i < a.B ? a.fresh[bt + i] : 0;
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            s[i] = plan_seq(a, c[i], f[i]);
            n += s[i].need;
            t += s[i].n;
        }
        const int64_t in = plan_wave_sum(n), it = plan_wave_sum(t);
        __syncthreads();  // the last round's sums have been read
        if (lane == 63) sm_n[wave] = in, sm_t[wave] = it;
        __syncthreads();
        int64_t on = cn + in - n, ot = ct + it - t;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < wave) on += sm_n[w], ot += sm_t[w];
            cn += sm_n[w], ct += sm_t[w];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int b = b0 + E * threadIdx.x + i;
            if (b < a.B) {
                off[b] = sat32(on), cu[b] = sat32(ot);
                if (cl) cl[b] = c[i], nl[b] = f[i];
                const bool fit = s[i].fit(on, a.F);
                refused += !fit;
                if (fit && s[i].need) taken = max(taken, (int)(on + s[i].need));
            }
            on += s[i].need;
            ot += s[i].n;
        }
    }
    if (report) {  // one LDS atomic a wave: one a sequence kept the first workgroup 8 us behind the others at 1024 sequences
        taken = wave_reduce(taken, [](int x, int y) { return max(x, y); }, 0);
        refused = wave_sum_i(refused);
        if (lane == 0) {
            atomicMax(&sh_taken, taken);
            atomicAdd(&sh_refused, refused);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        off[a.B] = sat32(cn);
        cu[a.B] = sat32(ct);
        if (report) {
            a.counts[0] = sat32(ct);
            a.counts[1] = sat32(cn);
            a.counts[2] = sh_taken;
            a.counts[3] = sh_refused;
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kPlanThreads) void k_page_plan_scan(PlanArgs a) { plan_scan<4>(a, a.ws_off, a.ws_cu, nullptr, nullptr, true); }

// the last b with at[b] <= v (at ascends, at[0] = 0, v < at[B])
__device__ __forceinline__ int plan_find(const int32_t* at, int B, int v) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// tokens t0 .. t0 + N - 1 (their sums and lengths in LDS or global memory)
template <int N>
__device__ __forceinline__ void plan_tokens(const PlanArgs& a, const int32_t* off, const int32_t* cu, const int32_t* cl, const int32_t* nl,
                                            int64_t t0) {
    int pg[N], sl[N], rw[N], ps[N];
    int b = t0 < cu[a.B] ? plan_find(cu, a.B, (int)t0) : -1, known = -1;
    int64_t o = 0;
    PlanSeq s{};
    bool fit = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t t = t0 + i;
        pg[i] = sl[i] = rw[i] = ps[i] = -1;
        if (t >= cu[a.B]) continue;  // behind the last sequence
        while (cu[b + 1] <= t) ++b;
        if (b != known) {
            s = plan_seq(a, cl[b], nl[b]);
            o = off[b];
            fit = s.fit(o, a.F);
            known = b;
        }
        const uint32_t pos = s.c + (uint32_t)(t - cu[b]);  // < c + n < 2^32
        rw[i] = b;
        ps[i] = sat32(pos);
        if (!fit) continue;
        const uint32_t blk = plan_div(a, pos);
        sl[i] = (int)(pos - blk * (uint32_t)a.page);
        if (i > 0 && sl[i] > 0 && rw[i - 1] == b) {  // the token before stands on the same page
            pg[i] = pg[i - 1];
        } else {
            const int32_t* at = blk < s.have ? a.table + b * a.ts + blk : a.free_pages + (o + blk - s.have);
            pg[i] = *at;
        }
    }
    if constexpr (N == 4) {
        if (t0 + 4 <= a.T) {  // the launch saw to the arrays' alignment
            *reinterpret_cast<int4*>(a.pages + t0) = make_int4(pg[0], pg[1], pg[2], pg[3]);
            *reinterpret_cast<int4*>(a.slots + t0) = make_int4(sl[0], sl[1], sl[2], sl[3]);
            *reinterpret_cast<int4*>(a.rows + t0) = make_int4(rw[0], rw[1], rw[2], rw[3]);
            *reinterpret_cast<int4*>(a.pos + t0) = make_int4(ps[0], ps[1], ps[2], ps[3]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (t0 + i >= a.T) break;
        a.pages[t0 + i] = pg[i];
        a.slots[t0 + i] = sl[i];
        a.rows[t0 + i] = rw[i];
        a.pos[t0 + i] = ps[i];
    }
}

// LDS: the sums in LDS, scanned here. N: tokens a thread takes.
template <bool LDS, int N>
__global__ __launch_bounds__(kPlanThreads) void k_page_plan(PlanArgs a) {
    __shared__ int32_t sm[LDS ? 4 * (kPlanLdsSeqs + 1) : 1];
    const int32_t *off = a.ws_off, *cu = a.ws_cu, *cl = a.cached, *nl = a.fresh;
    if constexpr (LDS) {
        constexpr int S = kPlanLdsSeqs + 1;
        if (a.B <= kPlanThreads) plan_scan<1>(a, sm, sm + S, sm + 2 * S, sm + 3 * S, blockIdx.x == 0);
        else plan_scan<4>(a, sm, sm + S, sm + 2 * S, sm + 3 * S, blockIdx.x == 0);
        off = sm, cu = sm + S, cl = sm + 2 * S, nl = sm + 3 * S;
    }
    const int me = blockIdx.x * kPlanThreads + threadIdx.x, all = gridDim.x * kPlanThreads;
    // the pages that are taken, one a thread: into their sequence's row
    for (int64_t i = me, n = min(off[a.B], a.F); i < n; i += all) {
        const int b = plan_find(off, a.B, (int)i);
        const PlanSeq s = plan_seq(a, cl[b], nl[b]);
        if (s.fit(off[b], a.F)) a.table[b * a.ts + s.have + (i - off[b])] = a.free_pages[i];
    }
    for (int b = me; b <= a.B; b += all) a.cu[b] = cu[b];
    if ((int64_t)me * N < a.T) plan_tokens<N>(a, off, cu, cl, nl, (int64_t)me * N);
}

template <bool LDS>
static void plan_launch(const PlanArgs& a, hipStream_t st) {
    const bool wide = a.T >= kPlanWide && aligned16(a.pages) && aligned16(a.slots) && aligned16(a.rows) && aligned16(a.pos);
    const int each = kPlanThreads * (wide ? 4 : 1);
    // a thread for every token (or four); at least a workgroup for every 512 sequences (the table's entries)
    const int grid = max(max((a.T + each - 1) / each, min((a.B + 511) / 512, 64)), 1);
    if (wide) hipLaunchKernelGGL((k_page_plan<LDS, 4>), dim3(grid), dim3(kPlanThreads), 0, st, a);
    else hipLaunchKernelGGL((k_page_plan<LDS, 1>), dim3(grid), dim3(kPlanThreads), 0, st, a);
}

}  // namespace wf

using namespace wf;

extern "C" {

int64_t wf_kv_page_plan_ws_bytes(int B) { return B > kPlanLdsSeqs ? 2 * ((int64_t)B + 1) * 4 : 0; }

int wf_kv_page_plan(const int32_t* cached_lens, const int32_t* new_lens, int B, const int32_t* free_pages, int num_free,
                    int32_t* page_table, int64_t table_stride, int max_blocks, int page_size, int num_tokens, int32_t* pages,
                    int32_t* slots, int32_t* rows, int32_t* positions, int32_t* cu_tokens, int32_t* counts, void* ws,
                    void* stream) {
    WF_REQUIRE(B >= 0 && num_free >= 0 && num_tokens >= 0, "kv_page_plan: negative size (B %d, free %d, tokens %d)", B, num_free,
               num_tokens);
    WF_REQUIRE(page_size > 0 && page_size <= 65536, "kv_page_plan: page_size %d not in [1, 65536]", page_size);
    WF_REQUIRE(max_blocks >= 0 && table_stride >= max_blocks, "kv_page_plan: table rows of %d entries at stride %lld", max_blocks,
               (long long)table_stride);
    WF_REQUIRE((int64_t)max_blocks * page_size <= 0x7fffffff, "kv_page_plan: table rows reach past position 2^31 - 1");
    WF_REQUIRE(cu_tokens && counts, "kv_page_plan: null cu_tokens / counts");
    WF_REQUIRE(B == 0 || (cached_lens && new_lens && (page_table || max_blocks == 0)), "kv_page_plan: null lengths / table");
    WF_REQUIRE(num_free == 0 || free_pages, "kv_page_plan: null free list");
    WF_REQUIRE(num_tokens == 0 || (pages && slots && rows && positions), "kv_page_plan: null token arrays");
    WF_REQUIRE(B <= 1 << 24, "kv_page_plan: too many sequences (%d)", B);
    WF_REQUIRE(num_tokens <= 0x7fffffff - 4096, "kv_page_plan: too many tokens (%d)", num_tokens);
    PlanArgs a{cached_lens, new_lens, B, free_pages, num_free, page_table, table_stride, max_blocks, page_size,
               page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size), num_tokens, pages, slots, rows, positions, cu_tokens, counts,
               nullptr, nullptr, aligned16(cached_lens) && aligned16(new_lens)};
    hipStream_t st = as_stream(stream);
    if (B <= kPlanLdsSeqs) {
        plan_launch<true>(a, st);
    } else {
        WF_REQUIRE(ws, "kv_page_plan: null workspace");
        a.ws_off = reinterpret_cast<int32_t*>(ws);
        a.ws_cu = a.ws_off + B + 1;
        hipLaunchKernelGGL(k_page_plan_scan, dim3(1), dim3(kPlanThreads), 0, st, a);
        plan_launch<false>(a, st);
    }
    return check_launch("kv_page_plan");
}

}  // extern "C"
