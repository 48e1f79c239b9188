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
#include "wf_common.h"
#include "wf_device.h"

namespace wf {

constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 4 * kPlanThreads;  // tokens a workgroup fills, four neighbours a thread
constexpr int kPlanLdsSeqs = 2048;             // two int32 arrays of this many + 1 in LDS (16 KiB)

struct PlanArgs {
    const int32_t *cached, *fresh;
    int B;
    const int32_t* free_pages;
    int F;
    int32_t* table;
    int64_t ts;
    int cols, page, T;
    int32_t *pages, *slots, *rows, *pos, *cu, *counts;
    int32_t *ws_off, *ws_cu;  // [B + 1] each, B > kPlanLdsSeqs only
    int vec;                  // the four token arrays are 16-byte aligned
};

// Lengths are clamped to >= 0; sums are 64 bits and saturate where they are stored as 32.
__device__ __forceinline__ int32_t sat32(int64_t v) { return (int32_t)(v < 0x7fffffff ? v : 0x7fffffff); }

struct PlanSeq {
    int64_t c, n;         // held and new tokens
    int64_t have, total;  // pages held, pages after
    bool lng;             // does not fit the table row
    __device__ __forceinline__ int64_t need() const { return lng ? 0 : total - have; }
    // pages [off, off + need) of the free list are there
    __device__ __forceinline__ bool fit(int64_t off, int F) const { return !lng && (need() == 0 || off + need() <= F); }
};
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int b) {
    PlanSeq s;
    s.c = max(a.cached[b], 0);
    s.n = max(a.fresh[b], 0);
    const uint32_t p = (uint32_t)a.page;
    s.have = ((uint32_t)s.c + (p - 1)) / p;  // c + p - 1 < 2^32
    // c + n may pass 2^32: quotients and remainders apart
    const uint32_t c = (uint32_t)s.c, n = (uint32_t)s.n;
    const uint32_t rem = c % p + n % p;
    s.total = (int64_t)(c / p) + n / p + (rem + p - 1) / p;
    s.lng = s.total > a.cols;
    return s;
}

// Exclusive sums of need and n over all sequences into off[0..B], cu[0..B]; thread t takes four
// neighbours of every 1024. Workgroup 0's call also leaves the counts.
__device__ void plan_scan(const PlanArgs& a, int32_t* off, int32_t* cu, bool report) {
    __shared__ int64_t sm_n[4], sm_t[4];
    __shared__ int sh_taken, sh_refused;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) sh_taken = sh_refused = 0;
    int64_t cn = 0, ct = 0;  // sums before this 1024
    for (int b0 = 0; b0 < a.B; b0 += kPlanTokens) {
        int64_t n4[4], t4[4], n = 0, t = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + 4 * threadIdx.x + i;
            n4[i] = t4[i] = 0;
            if (b < a.B) {
                const PlanSeq s = plan_seq(a, b);
                n4[i] = s.need();
                t4[i] = s.n;
            }
            n += n4[i];
            t += t4[i];
        }
        int64_t in = n, it = t;  // inclusive over the wave
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t un = __shfl_up(in, d, 64), ut = __shfl_up(it, d, 64);
            if (lane >= d) in += un, it += ut;
        }
        __syncthreads();  // the last round's sums have been read
        if (lane == 63) sm_n[wave] = in, sm_t[wave] = it;
        __syncthreads();
        int64_t on = cn + in - n, ot = ct + it - t;
        for (int w = 0; w < wave; ++w) on += sm_n[w], ot += sm_t[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + 4 * threadIdx.x + i;
            if (b < a.B) off[b] = sat32(on), cu[b] = sat32(ot);
            if (report && b < a.B) {
                const PlanSeq s = plan_seq(a, b);
                if (!s.fit(on, a.F)) atomicAdd(&sh_refused, 1);
                else if (n4[i]) atomicMax(&sh_taken, (int)(on + n4[i]));
            }
            on += n4[i];
            ot += t4[i];
        }
        for (int w = 0; w < 4; ++w) cn += sm_n[w], ct += sm_t[w];
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

__global__ __launch_bounds__(kPlanThreads) void k_page_plan_scan(PlanArgs a) { plan_scan(a, a.ws_off, a.ws_cu, true); }

template <bool LDS>
__global__ __launch_bounds__(kPlanThreads) void k_page_plan(PlanArgs a) {
    __shared__ int32_t sm[LDS ? 2 * (kPlanLdsSeqs + 1) : 1];
    const int32_t *off = a.ws_off, *cu = a.ws_cu;
    if constexpr (LDS) {
        plan_scan(a, sm, sm + kPlanLdsSeqs + 1, blockIdx.x == 0);
        off = sm, cu = sm + kPlanLdsSeqs + 1;
    }
    // the table rows, a wave per sequence: entries [have, total) only
    for (int b = blockIdx.x * 4 + (threadIdx.x >> 6); b < a.B; b += gridDim.x * 4) {
        const PlanSeq s = plan_seq(a, b);
        const int64_t o = off[b];
        if (!s.fit(o, a.F)) continue;
        for (int64_t i = threadIdx.x & 63; i < s.need(); i += 64) a.table[b * a.ts + s.have + i] = a.free_pages[o + i];
    }
    for (int b = blockIdx.x * kPlanThreads + threadIdx.x; b <= a.B; b += gridDim.x * kPlanThreads) a.cu[b] = cu[b];
    // the tokens: four neighbours a thread
    const int64_t t0 = (int64_t)blockIdx.x * kPlanTokens + 4 * threadIdx.x;
    if (t0 >= a.T) return;
    int lo = 0, hi = a.B;  // the last b with cu[b] <= t0 (cu[0] = 0)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t0) lo = mid;
        else hi = mid;
    }
    int b = lo, pg[4], sl[4], rw[4], ps[4];
    int64_t o = 0;
    PlanSeq s;
    bool fit = false;
    int known = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + i;
        pg[i] = sl[i] = rw[i] = ps[i] = -1;
        if (t >= cu[a.B]) continue;  // behind the last sequence (also B == 0)
        while (cu[b + 1] <= t) ++b;
        if (b != known) {
            s = plan_seq(a, b);
            o = off[b];
            fit = s.fit(o, a.F);
            known = b;
        }
        const int64_t pos = s.c + (t - cu[b]);
        rw[i] = b;
        ps[i] = sat32(pos);
        if (!fit) continue;
        const uint32_t blk = (uint32_t)pos / (uint32_t)a.page;  // fits the row: pos < cols * page
        sl[i] = (int)((uint32_t)pos - blk * (uint32_t)a.page);
        pg[i] = blk < s.have ? a.table[b * a.ts + blk] : a.free_pages[o + blk - s.have];
    }
    if (a.vec && t0 + 4 <= a.T) {
        *reinterpret_cast<int4*>(a.pages + t0) = make_int4(pg[0], pg[1], pg[2], pg[3]);
        *reinterpret_cast<int4*>(a.slots + t0) = make_int4(sl[0], sl[1], sl[2], sl[3]);
        *reinterpret_cast<int4*>(a.rows + t0) = make_int4(rw[0], rw[1], rw[2], rw[3]);
        *reinterpret_cast<int4*>(a.pos + t0) = make_int4(ps[0], ps[1], ps[2], ps[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (t0 + i >= a.T) break;
        a.pages[t0 + i] = pg[i];
        a.slots[t0 + i] = sl[i];
        a.rows[t0 + i] = rw[i];
        a.pos[t0 + i] = ps[i];
    }
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
    WF_REQUIRE(num_tokens <= 0x7fffffff - kPlanTokens, "kv_page_plan: too many tokens");
    PlanArgs a{cached_lens, new_lens, B, free_pages, num_free, page_table, table_stride, max_blocks, page_size, num_tokens, pages,
               slots, rows, positions, cu_tokens, counts, nullptr, nullptr,
               aligned16(pages) && aligned16(slots) && aligned16(rows) && aligned16(positions)};
    // at least a workgroup for every 1024 tokens; the table rows spread over up to 256
    const int grid = max(max((num_tokens + kPlanTokens - 1) / kPlanTokens, min((B + 63) / 64, 256)), 1);
    hipStream_t st = as_stream(stream);
    if (B <= kPlanLdsSeqs) {
        hipLaunchKernelGGL((k_page_plan<true>), dim3(grid), dim3(kPlanThreads), 0, st, a);
    } else {
        WF_REQUIRE(ws, "kv_page_plan: null workspace");
        a.ws_off = reinterpret_cast<int32_t*>(ws);
        a.ws_cu = a.ws_off + B + 1;
        hipLaunchKernelGGL(k_page_plan_scan, dim3(1), dim3(kPlanThreads), 0, st, a);
        hipLaunchKernelGGL((k_page_plan<false>), dim3(grid), dim3(kPlanThreads), 0, st, a);
    }
    return check_launch("kv_page_plan");
}

}  // extern "C"
