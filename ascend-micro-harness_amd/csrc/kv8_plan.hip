// kv8_plan.hip -- the page plan of a serving step (tq4_paged_plan, tq4_kv8.h).
//
// Three prefix sums over the requests decide everything: the new tokens (row
// ranges), the pages wanted by requests that fit (which are granted, and where
// in the ring their pages lie) and the pages given back. Every table entry,
// slot and position then follows from its request's six numbers, so the rest
// is independent stores. A token's page is the ring's entry when the call opens
// it and the table's otherwise, so slots need not wait for the tables.
//
// Latency bounds it: a round trip for the lengths, the scans, one for the table
// or ring entries, the stores. So one launch where it can be: each workgroup
// makes the scans for itself (a thread a request, the records in LDS) and fills
// its share of rows and tables. 64 requests 4.5 us, 1000 with 61000 rows 8.0 (three
// launches: 12; in place, in two: 15); 0.55 MB, so a launch is the floor of both.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_device.hpp"

namespace tq4 {
namespace {

using kv8::div_by;
using kv8::Divisor;
using kv8::wave_scan;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kHeld = 2048;            // requests whose records lie in LDS
constexpr uint32_t kRowsPerBlock = 2048;
constexpr uint32_t kAloneRows = 4096;       // rows that one workgroup fills in place

// What the scans leave of a request for the fill.
struct Request {
    uint32_t first;  // its first row
    uint32_t rows;   // its rows when granted, else 0
    uint32_t base;   // tokens in its cache before them
    uint32_t pop;    // its first opened page's place in the ring's taken run
    uint32_t back;   // pages it gives back
    uint32_t push;   // the first of them's place in the ring's returned run
};

struct Ring {
    uint32_t head, count;
};

struct Pages {
    Divisor per_page;  // tokens of a page
    uint32_t S, P;

    __device__ __forceinline__ uint32_t of(uint32_t tokens) const  // ceil(tokens / S)
    {
        const uint32_t q = div_by(tokens, per_page);
        return q + (q * S < tokens ? 1u : 0u);
    }
    // the ring's entry `offset` (at most P) behind its head
    __device__ __forceinline__ uint32_t at(const Ring& r, uint32_t offset) const
    {
        const uint64_t i = (uint64_t)r.head + offset;
        return (uint32_t)(i < P ? i : i - P);
    }
};

// Inclusive sum over the workgroup; `total` the whole. part: kWaves words of LDS
// that nothing else uses up to the next barrier.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if (lane == 63u) part[wave] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint64_t x = part[w];
        all += x;
        if ((uint32_t)w < wave) before += x;
    }
    total = all;
    return v + before;
}

struct ScanLds {
    uint64_t part[2][kWaves];
    uint32_t taken;
};

// The scans: the requests' records to rec. `writes`: the workgroup that stores
// the row ranges, the granted rows, the new lengths and the ring's new state. In
// place is allowed for the last two (in a launch of one workgroup): a thread
// reads what it overwrites, the state is read before a barrier.
__device__ __forceinline__ Ring scan_requests(const PlanParams& p, const Pages& pages,
                                              Request* rec, ScanLds& lds, bool writes)
{
    const uint64_t room = (uint64_t)p.M * p.S;
    const uint32_t cap = room < 0x7fffffffull ? (uint32_t)room : 0x7fffffffu;
    const int32_t head = p.state[0] % (int32_t)p.P, count = p.state[1];
    Ring r;
    r.head = (uint32_t)(head < 0 ? head + (int32_t)p.P : head);
    r.count = count < 0 ? 0u : (uint32_t)count > p.P ? p.P : (uint32_t)count;
    if (threadIdx.x == 0) lds.taken = 0;
    uint64_t tokens = 0, both = 0;  // both: pages wanted, and given back above them
    for (uint32_t b0 = 0; b0 < p.B; b0 += kThreads) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t c = 0, n = 0;
        bool leaves = false;
        if (b < p.B) {
            const int32_t ci = p.context_lens[b], ni = p.query_lens[b];
            leaves = p.release && p.release[b] != 0;
            c = ci < 0 ? 0u : (uint32_t)ci > cap ? cap : (uint32_t)ci;
            n = ni < 0 ? 0u : (uint32_t)ni;
        }
        const uint32_t base = leaves ? 0u : c, back = leaves ? pages.of(c) : 0u;
        uint64_t sum;
        const uint64_t to = tokens + block_scan(n, lds.part[0], sum);
        tokens += sum;
        // (base + n < 2^32; beyond 2^31 it does not fit)
        const bool fits = b < p.B && base + n <= cap && to <= p.T;
        const uint32_t want = fits ? pages.of(base + n) - pages.of(base) : 0u;
        const uint64_t upto = both + block_scan((uint64_t)back << 32 | want, lds.part[1], sum);
        both += sum;
        const uint32_t wanted = (uint32_t)upto, given = (uint32_t)(upto >> 32);
        const bool ok = fits && (want == 0 || wanted <= r.count);
        if (ok && want) atomicMax(&lds.taken, wanted);
        if (b < p.B) {
            const uint64_t from = to - n;
            Request q;
            q.first = from < 0x7fffffffull ? (uint32_t)from : 0x7fffffffu;
            q.rows = ok ? n : 0u;
            q.base = base;
            q.pop = ok ? wanted - want : 0u;
            q.back = back;
            q.push = given - back;
            rec[b] = q;
            if (writes) {
                if (b == 0) p.cu[0] = 0;
                p.cu[b + 1] = to < 0x7fffffffull ? (int32_t)to : 0x7fffffff;
                p.granted[b] = (int32_t)q.rows;
                p.new_lens[b] = (int32_t)(base + q.rows);
            }
        }
    }
    __syncthreads();
    if (writes && threadIdx.x == 0) {
        const uint32_t taken = lds.taken;
        const uint64_t left = (uint64_t)r.count - taken + (both >> 32);
        p.new_state[0] = (int32_t)pages.at(r, taken);
        p.new_state[1] = (int32_t)(left < p.P ? left : p.P);
    }
    return r;
}

// The table entries that a request's numbers change: [begin, end).
struct Entries {
    uint32_t begin, held, opened, end;

    __device__ __forceinline__ Entries(const Pages& pages, const Request& q)
    {
        held = pages.of(q.base);
        opened = pages.of(q.base + q.rows);
        // [0, back) are read, [held, opened) written; a request that gives pages
        // back holds none, so both begin at 0 then
        begin = q.back ? 0u : held;
        end = q.back > opened ? q.back : opened;
    }
};

// Entry i of request b: a page that it gives back goes to the ring's end, then
// the page that it opens comes from the head. One lane reads and writes an entry;
// the returned run lies behind the `count` entries that the opened pages are read
// from, or is dropped.
__device__ __forceinline__ void fill_entry(const PlanParams& p, const Pages& pages, const Ring& r,
                                           const Request& q, const Entries& e, uint32_t b,
                                           uint32_t i)
{
    int32_t* at = p.tables + (uint64_t)b * p.M + i;
    if (i < q.back) {
        const uint64_t to = (uint64_t)r.count + q.push + i;
        if (to < p.P) p.ring[pages.at(r, (uint32_t)to)] = *at;
    }
    if (i >= e.held && i < e.opened) *at = p.ring[pages.at(r, q.pop + (i - e.held))];
}

// A wave's requests [b0, b0 + count), at most 64: a lane each where the entries
// are few (a decode step), the whole wave in turn for the others.
__device__ __forceinline__ void fill_tables(const PlanParams& p, const Pages& pages, const Ring& r,
                                            const Request* rec, uint32_t b0, uint32_t count)
{
    constexpr uint32_t kFew = 2;
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t many = 0;
    if (lane < count) {
        const Request q = rec[b0 + lane];
        const Entries e(pages, q);
        many = e.end > e.begin + kFew ? 1u : 0u;
        if (!many)
            for (uint32_t i = e.begin; i < e.end; ++i) fill_entry(p, pages, r, q, e, b0 + lane, i);
    }
    uint64_t rest = __ballot(many);
    while (rest) {
        const uint32_t b = b0 + (uint32_t)__builtin_ctzll(rest);
        rest &= rest - 1;
        const Request q = rec[b];
        const Entries e(pages, q);
        for (uint32_t i = e.begin + lane; i < e.end; i += 64) fill_entry(p, pages, r, q, e, b, i);
    }
}

// Row t of the step. Its request is the last whose first row is at or before t:
// of several with that first row all but the last have no rows.
__device__ __forceinline__ void fill_row(const PlanParams& p, const Pages& pages, const Ring& r,
                                         const Request* rec, uint32_t t)
{
    uint32_t lo = 0, hi = p.B;  // the first request with first > t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (rec[mid].first > t) hi = mid;
        else lo = mid + 1;
    }
    int32_t slot = -1, pos = 0;
    if (lo > 0) {
        const Request q = rec[lo - 1];
        const uint32_t off = t - q.first;
        if (off < q.rows) {
            const uint32_t at = q.base + off, i = div_by(at, pages.per_page);
            const uint32_t held = pages.of(q.base);
            const int32_t page = i >= held ? p.ring[pages.at(r, q.pop + (i - held))]
                                           : p.tables[(uint64_t)(lo - 1) * p.M + i];
            pos = (int32_t)at;
            if (page >= 0 && (uint32_t)page < p.P)
                slot = (int32_t)((uint32_t)page * p.S + (at - i * p.S));
        }
    }
    p.slots[t] = slot;
    if (p.positions) p.positions[t] = pos;
}

__device__ __forceinline__ void fill(const PlanParams& p, const Pages& pages, const Ring& r,
                                     const Request* rec, uint32_t block, uint32_t blocks)
{
    for (uint32_t t = block * kThreads + threadIdx.x; t < p.T; t += blocks * kThreads)
        fill_row(p, pages, r, rec, t);
    uint32_t each = (p.B + blocks * kWaves - 1) / (blocks * kWaves);
    if (each > 64) each = 64;
    for (uint32_t b = (block * kWaves + (threadIdx.x >> 6)) * each; b < p.B;
         b += blocks * kWaves * each)
        fill_tables(p, pages, r, rec, b, p.B - b < each ? p.B - b : each);
}

// Scans and fill in one launch, of one workgroup where lengths or state are in
// place.
__global__ __launch_bounds__(kThreads) void plan_step(PlanParams p, Pages pages)
{
    __shared__ Request rec[kHeld];
    __shared__ ScanLds lds;
    const Ring r = scan_requests(p, pages, rec, lds, blockIdx.x == 0);
    fill(p, pages, r, rec, blockIdx.x, gridDim.x);
}

// The same in two launches, the records in the workspace, behind the ring's state.
__global__ __launch_bounds__(kThreads) void plan_scan(PlanParams p, Pages pages)
{
    __shared__ ScanLds lds;
    const Ring r = scan_requests(p, pages, (Request*)(p.ws + 2), lds, true);
    if (threadIdx.x == 0) *(Ring*)p.ws = r;
}

__global__ __launch_bounds__(kThreads) void plan_fill(PlanParams p, Pages pages)
{
    fill(p, pages, *(const Ring*)p.ws, (const Request*)(p.ws + 2), blockIdx.x, gridDim.x);
}

}  // namespace

size_t plan_workspace_bytes(uint32_t B) { return sizeof(Ring) + (size_t)B * sizeof(Request); }

hipError_t launch_plan(hipStream_t stream, const PlanParams& p)
{
    Pages pages;
    pages.per_page = kv8::div_magic(p.S);
    pages.S = p.S;
    pages.P = p.P;
    // workgroups: a tile of rows each, 256 requests at most
    uint32_t blocks = (p.T + kRowsPerBlock - 1) / kRowsPerBlock;
    const uint32_t by_requests = (p.B + 255) / 256;
    if (blocks < by_requests) blocks = by_requests;
    if (blocks > 1024) blocks = 1024;
    const bool in_place = p.new_lens == p.context_lens || p.new_state == p.state;
    if (p.B <= kHeld && (!in_place || p.T <= kAloneRows)) {
        hipLaunchKernelGGL(plan_step, dim3(in_place ? 1 : blocks), dim3(kThreads), 0, stream, p,
                           pages);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(plan_scan, dim3(1), dim3(kThreads), 0, stream, p, pages);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(plan_fill, dim3(blocks), dim3(kThreads), 0, stream, p, pages);
    return hipGetLastError();
}

}  // namespace tq4
