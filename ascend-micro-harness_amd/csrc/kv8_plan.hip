// kv8_plan.hip -- the page plan of a serving step (tq4_paged_plan, tq4_kv8.h).
//
// Three prefix sums over the requests decide everything: the new tokens (row
// ranges), the pages wanted by requests that fit (which are granted, and where
// in the ring their pages lie) and the pages given back. Every table entry,
// slot and position then follows from its request's five numbers, so the rest
// is independent stores. A token's page is the ring's entry when the call opens
// it and the table's otherwise, so slots need not wait for the tables.
//
// Latency bounds it (546 KB for 1000 requests of a mixed batch): a round trip
// for the lengths, the scans, one for the table or ring entries, the stores.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_internal.hpp"

namespace tq4 {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanWaves = kScanThreads / 64;
constexpr int kFillThreads = 256;
constexpr uint32_t kTokensPerBlock = 1024;

// What the scan leaves of a request for the fill.
struct Request {
    int32_t base;    // tokens in its cache before the new ones
    int32_t want;    // pages it opens (0 when not granted)
    uint32_t pop;    // its first page's place in the ring's taken run
    int32_t back;    // pages it gives back
    uint32_t push;   // its first page's place in the ring's returned run
    int32_t first;   // its first row
    int32_t rows;    // its rows when granted, else 0
    int32_t pad;
};
static_assert(sizeof(Request) == 32, "two 16-byte loads");

struct Header {
    uint32_t head, count;
    uint32_t pad[6];
};
static_assert(sizeof(Header) == 32, "keeps the requests aligned");

// Inclusive sum over the workgroup; `total` the whole sum. part: kScanWaves
// words of LDS, free again after the call's second barrier.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint64_t o = __shfl_up(v, s);
        if (lane >= (uint32_t)s) v += o;
    }
    __syncthreads();
    if (lane == 63u) part[wave] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) {
        const uint64_t x = part[w];
        all += x;
        if ((uint32_t)w < wave) before += x;
    }
    total = all;
    return v + before;
}

__device__ __forceinline__ uint32_t ring_at(const Header& h, uint32_t P, uint64_t offset)
{
    return (uint32_t)((h.head + offset) % P);
}

// The scans: requests' records to `rec`, the row ranges, the granted rows, the
// new lengths and the ring's new state. In place is allowed for the last two:
// a thread reads what it overwrites, the state is read before a barrier.
__device__ __forceinline__ void scan_requests(const PlanParams& p, Header* hdr, Request* rec,
                                              uint64_t* part)
{
    const int64_t cap = (int64_t)p.M * p.S < 0x7fffffffll ? (int64_t)p.M * p.S : 0x7fffffffll;
    Header h{};
    int32_t head = p.state[0], count = p.state[1];
    head = head % (int32_t)p.P;
    h.head = (uint32_t)(head < 0 ? head + (int32_t)p.P : head);
    h.count = count < 0 ? 0u : (uint32_t)count > p.P ? p.P : (uint32_t)count;
    uint64_t tokens = 0, wanted = 0, backs = 0, taken = 0;
    for (uint32_t b0 = 0; b0 < p.B; b0 += kScanThreads) {
        const uint32_t b = b0 + threadIdx.x;
        int64_t c = 0, n = 0;
        bool leaves = false;
        if (b < p.B) {
            c = p.context_lens[b];
            n = p.query_lens[b];
            leaves = p.release && p.release[b] != 0;
            c = c < 0 ? 0 : c > cap ? cap : c;
            n = n < 0 ? 0 : n;
        }
        const int64_t base = leaves ? 0 : c;
        const uint32_t back = leaves ? (uint32_t)((c + p.S - 1) / p.S) : 0u;
        uint64_t sum;
        const uint64_t to = tokens + block_scan((uint64_t)n, part, sum);
        tokens += sum;
        const bool fits = b < p.B && base + n <= cap && to <= p.T;
        const uint32_t want =
            fits ? (uint32_t)((base + n + p.S - 1) / p.S - (base + p.S - 1) / p.S) : 0u;
        const uint64_t upto = wanted + block_scan(want, part, sum);
        wanted += sum;
        const uint64_t given = backs + block_scan(back, part, sum);
        backs += sum;
        const bool ok = fits && (want == 0 || upto <= h.count);
        block_scan(ok ? want : 0u, part, sum);
        taken += sum;
        if (b < p.B) {
            const uint64_t from = to - (uint64_t)n;
            if (b == 0) p.cu[0] = 0;
            p.cu[b + 1] = to < 0x7fffffffull ? (int32_t)to : 0x7fffffff;
            p.granted[b] = ok ? (int32_t)n : 0;
            p.new_lens[b] = (int32_t)(ok ? base + n : base);
            Request r;
            r.base = (int32_t)base;
            r.want = ok ? (int32_t)want : 0;
            r.pop = ok ? (uint32_t)(upto - want) : 0u;
            r.back = (int32_t)back;
            r.push = (uint32_t)(given - back < p.P ? given - back : p.P);
            r.first = from < 0x7fffffffull ? (int32_t)from : 0x7fffffff;
            r.rows = ok ? (int32_t)n : 0;
            r.pad = 0;
            rec[b] = r;
        }
    }
    if (threadIdx.x == 0) {
        *hdr = h;
        // (the last scan's barriers lie behind every thread's read of the state)
        const uint64_t left = h.count - taken + backs;
        p.new_state[0] = (int32_t)((h.head + taken) % p.P);
        p.new_state[1] = (int32_t)(left < p.P ? left : p.P);
    }
}

// Request b's table entries, a thread each: the pages it gives back go to the
// ring's end, then the pages it opens come from the head. One thread reads and
// writes an entry; the returned run lies behind the `count` entries that the
// opened pages are read from, or is dropped.
__device__ __forceinline__ void fill_pages(const PlanParams& p, const Header& h, const Request& r,
                                           uint32_t b, uint32_t thread, uint32_t threads)
{
    const uint32_t held = (uint32_t)(((int64_t)r.base + p.S - 1) / p.S);
    const uint32_t opened = held + (uint32_t)r.want;
    int32_t* row = p.tables + (uint64_t)b * p.M;
    // entries [0, back) are read, [held, opened) written; a request that gives
    // pages back holds none, so both begin at 0 then
    const uint32_t end = (uint32_t)r.back > opened ? (uint32_t)r.back : opened;
    for (uint32_t i = (r.back > 0 ? 0u : held) + thread; i < end; i += threads) {
        if (i < (uint32_t)r.back) {
            const uint64_t at = (uint64_t)h.count + r.push + i;
            if (at < p.P) p.ring[ring_at(h, p.P, at)] = row[i];
        }
        if (i >= held && i < opened)
            row[i] = p.ring[ring_at(h, p.P, (uint64_t)r.pop + (i - held))];
    }
}

// Row t of the step: its request is the last whose first row is at or before t
// among those with rows there.
__device__ __forceinline__ void fill_token(const PlanParams& p, const Header& h,
                                           const Request* rec, uint32_t t)
{
    uint32_t lo = 0, hi = p.B;  // the first request with first > t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((uint32_t)rec[mid].first > t) hi = mid;
        else lo = mid + 1;
    }
    // requests without rows that begin at t follow the one that owns t only if
    // they come later with the same first row: the last one with first <= t
    // owns t exactly when it has rows
    int32_t slot = -1, pos = 0;
    if (lo > 0) {
        const Request r = rec[lo - 1];
        const uint32_t off = t - (uint32_t)r.first;
        if (off < (uint32_t)r.rows) {
            pos = r.base + (int32_t)off;
            const uint32_t i = (uint32_t)pos / p.S;
            const uint32_t held = (uint32_t)(((int64_t)r.base + p.S - 1) / p.S);
            const int32_t page =
                i >= held ? p.ring[ring_at(h, p.P, (uint64_t)r.pop + (i - held))]
                          : p.tables[(uint64_t)(lo - 1) * p.M + i];
            if (page >= 0 && (uint32_t)page < p.P)
                slot = (int32_t)((uint32_t)page * p.S + ((uint32_t)pos - i * p.S));
        }
    }
    p.slots[t] = slot;
    if (p.positions) p.positions[t] = pos;
}

__global__ __launch_bounds__(kScanThreads) void plan_scan(PlanParams p)
{
    __shared__ uint64_t part[kScanWaves];
    scan_requests(p, (Header*)p.ws, (Request*)p.ws + 1, part);
}

__global__ __launch_bounds__(kFillThreads) void plan_fill(PlanParams p, uint32_t token_blocks)
{
    const Header h = *(const Header*)p.ws;
    const Request* rec = (const Request*)p.ws + 1;
    if (blockIdx.x < token_blocks) {
        const uint32_t t0 = blockIdx.x * kTokensPerBlock;
        for (uint32_t k = threadIdx.x; k < kTokensPerBlock && t0 + k < p.T; k += kFillThreads)
            fill_token(p, h, rec, t0 + k);
        return;
    }
    // a wave a request
    const uint32_t b = (blockIdx.x - token_blocks) * (kFillThreads / 64) + (threadIdx.x >> 6);
    if (b < p.B) fill_pages(p, h, rec[b], b, threadIdx.x & 63u, 64);
}

}  // namespace

size_t plan_workspace_bytes(uint32_t B) { return sizeof(Header) + (size_t)B * sizeof(Request); }

hipError_t launch_plan(hipStream_t stream, const PlanParams& p)
{
    hipLaunchKernelGGL(plan_scan, dim3(1), dim3(kScanThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint32_t token_blocks = (p.T + kTokensPerBlock - 1) / kTokensPerBlock;
    const uint32_t page_blocks = (p.B + kFillThreads / 64 - 1) / (kFillThreads / 64);
    hipLaunchKernelGGL(plan_fill, dim3(token_blocks + page_blocks), dim3(kFillThreads), 0, stream,
                       p, token_blocks);
    return hipGetLastError();
}

}  // namespace tq4
