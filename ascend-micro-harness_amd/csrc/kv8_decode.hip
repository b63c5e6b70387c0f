// kv8_decode.hip -- attention of few rows a sequence over the 8-bit paged cache
// (tq4_kv8_paged_decode, and tq4_kv8_paged_prefill of few rows; tq4_kv8.h).
//
// Up to 16 rows (the GQA group's heads, times the query tokens) of a (sequence,
// kv head) share a pass over its tokens. A wave takes 64 tokens, four strips, at
// a time:
//   S = K Q^T     MFMA 16x16x32 f16, tokens x rows. Codes are exact in f16 and a
//                 row of q is shifted by a power of two into f16's range.
//   s' = S * (k scale * q factor)                      log2 units
//   P = 2^(s' + log2(v scale) - m), in f16 with the v scale inside it, so the row's
//       largest product is 2^6 whatever the scales' spread; m moves when a row
//       passes 2^14 (lazily), and the sums with it
//   O^T += V^T P^T   on V's codes;  l += 2^(s' - s), as P times a strip's factor, where
//       s moves like m (References): weights whose products round to 0 count in l
//   out = O 2^m / (l 2^s)
// Tile j of S holds tokens 4j .. 4j + 3 of each of the four strips, so a lane's
// 16 scores are the 16 tokens of one strip (one scale each) for one row: they are
// the P^T operand as they lie, and the V^T operand is a channel's 16 consecutive
// bytes of that strip. Row factors are lane values; only the lazy maximum
// crosses lanes. The statistics and sums are 32-bit, held per wave and merged
// through LDS, then through records where a sequence is split. P is rounded to f16
// (2^-11 relative) and v's codes are exact in it; out is rounded once.
//
// The cache's bytes bound it, then the second kernel: 64 sequences of 512..8192
// tokens (552 MB) 109 us, 5.05 TB/s of 5.6 that reading the strips alone reaches; one
// of 65536 tokens of 2 heads of 256 (67 MB) 18 us and 6 to join 128 parts; one of
// 4096 6 and 4. A unit of 64 tokens keeps a lane's loads 16 bytes wide and a
// strip's scale one a lane; the loads run a unit ahead in the registers that the
// products just freed (a second set of registers spills at 256 channels).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_device.hpp"

namespace tq4 {
namespace {

using namespace kv8;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRows = 16;   // rows of a tile
constexpr int kUnit = 64;   // tokens of a wave's step
static_assert(kUnit == kKv8Unit && kRows == kKv8Rows, "the host sizes records and quotas by them");

// The block-table entries behind a unit: of the strip whose keys the lane loads
// and of the strip whose values it loads; -1 past the table.
struct Entries {
    int32_t k, v;
};

// Where a unit's bytes lie, and what of them is alive.
struct Place {
    const uint8_t *k, *v;
    float ks, vs;  // the scales of the lane's strip
    int live;      // its live tokens
};

template <int D>
struct Walk {
    const Kv8AttnParams* pp;
    const int32_t* table;
    Divisor per_page;   // strips of a page
    uint32_t h, L;
    uint32_t c, g;

    __device__ __forceinline__ int32_t entry(uint32_t strip) const
    {
        const Kv8AttnParams& p = *pp;
        const uint32_t i = div_by(strip, per_page);
        const int32_t e = table[i < p.M ? i : p.M - 1];
        return i < p.M ? e : -1;
    }
    __device__ __forceinline__ Entries entries(uint32_t t0) const
    {
        return {entry(t0 / 16 + (c >> 2)), entry(t0 / 16 + g)};
    }
    __device__ __forceinline__ uint32_t in_page(uint32_t strip) const
    {
        return strip - div_by(strip, per_page) * (pp->S / 16);
    }
    __device__ __forceinline__ Place place(uint32_t t0, Entries e) const
    {
        const Kv8AttnParams& p = *pp;
        const uint32_t sk = t0 / 16 + (c >> 2), sv = t0 / 16 + g;
        const bool ok = e.v >= 0 && (uint32_t)e.v < p.P;
        const uint32_t pk = e.k >= 0 && (uint32_t)e.k < p.P ? (uint32_t)e.k : 0u;
        const uint32_t pv = ok ? (uint32_t)e.v : 0u;
        const uint64_t rk = (uint64_t)pk * p.Hkv + h, rv = (uint64_t)pv * p.Hkv + h;
        Place x;
        x.k = p.key_cache + (rk * p.S + in_page(sk) * 16u + (c & 3u)) * D + 16u * g;
        x.v = p.value_cache + (rv * p.S + in_page(sv) * 16u) * D + 16u * c;
        x.ks = p.scales[rv];
        x.vs = p.scales[(uint64_t)p.P * p.Hkv + rv];
        const int left = (int)L - (int)(16u * sv);
        x.live = !ok || left < 0 ? 0 : left > 16 ? 16 : left;
        return x;
    }
};

// Keys and values of a unit as they come from memory.
template <int D>
struct KeyBytes {
    u4_t x[4][D / 64];  // tile, 64 channels

    __device__ __forceinline__ void fetch(const uint8_t* k)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) x[j][i] = *(const u4_t*)(k + 4 * j * D + 64 * i);
    }
};
template <int D>
struct ValueBytes {
    u4_t x[D / 16];  // 16 channels

    __device__ __forceinline__ void fetch(const uint8_t* v)
    {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) x[i] = *(const u4_t*)(v + 256 * i);
    }
};

struct Sequence : SequenceBase {
    __device__ __forceinline__ Sequence() {}
    __device__ __forceinline__ Sequence(const Kv8AttnParams& p, uint32_t b) : SequenceBase(p, b) {}
    // An item is a (sequence, kv head, tile of 16 rows); its units of 64 tokens:
    // one at least, which writes the zeros of rows that see nothing.
    __device__ __forceinline__ uint32_t units() const
    {
        return tokens ? (tokens + kUnit - 1) / kUnit : 1u;
    }
    __device__ __forceinline__ uint32_t tiles(const Kv8AttnParams& p) const
    {
        return (rows * p.G + kRows - 1) / kRows;
    }
    __device__ __forceinline__ uint32_t work(const Kv8AttnParams& p) const
    {
        return units() * tiles(p) * p.Hkv;
    }
    __device__ __forceinline__ Sequence of_lane(uint32_t lane) const
    {
        Sequence s;
        static_cast<SequenceBase&>(s) = SequenceBase::of_lane(lane);
        return s;
    }
};

// How a call is cut.
//  - Streamed (K = 0): the items' units lie on one line, sequence by sequence, and
//    workgroup w takes the `quota` units from w * quota on, so that all finish
//    together whatever the lengths are. An item that lies in several workgroups
//    leaves a record in each: slot 2w + 1 of the one that it begins in, 2w of those
//    behind it.
//  - K parts an item, whatever else is in the batch (a row's bits then do not
//    depend on its neighbours): slot item * K + part.
__device__ __forceinline__ uint32_t quota_of(const Kv8AttnParams& p, uint32_t total)
{
    const uint32_t q = ((total + p.groups - 1) / p.groups + kWaves - 1) / kWaves * kWaves;
    return q ? q : kWaves;  // a unit a wave at least
}
__device__ __forceinline__ uint32_t part_units(const Kv8AttnParams& p, uint32_t units)
{
    return (units + p.K - 1) / p.K;
}

// Part of an item, a workgroup's: units [begin, end), a record's slot, or -1 where
// it is the whole item.
struct Part {
    Sequence seq;
    uint32_t b, h, rt, begin, end;
    int64_t slot;
};

// What a lane knows of a part: its row, the tokens that the row sees, and its own
// walk over the pages.
template <int D>
struct Lane {
    Walk<D> walk;
    const uint16_t* q;  // the row's channels from the lane's on
    uint32_t first, units;
    int32_t limit;     // tokens that the row sees

    __device__ __forceinline__ Lane(const Kv8AttnParams& p, Divisor per_page, const Part& x)
        : walk{&p, p.tables + (uint64_t)x.b * p.M, per_page, x.h, x.seq.tokens, threadIdx.x & 15u,
               (threadIdx.x & 63u) >> 4}
    {
        // tokens that no row of the tile sees are left out. Those that some rows see and
        // others do not are fewer than kRows, in the last two units: a wave's last.
        uint32_t end = x.end;
        if (p.causal) {
            const uint32_t last = x.rt * kRows + kRows - 1, rows = x.seq.rows * p.G;
            walk.L = sees(x, (last < rows ? last : rows - 1) / p.G);
            const uint32_t units = (walk.L + kUnit - 1) / kUnit;
            end = end < units ? end : units;
        }
        const uint32_t wave = threadIdx.x >> 6, from = x.begin + wave;
        first = from * kUnit;
        units = from < end ? (end - from + kWaves - 1) / kWaves : 0u;
        // flat row f of the tile is token f / G, head f % G
        const uint32_t f = x.rt * kRows + walk.c, qi = f / p.G;
        const bool live = f < x.seq.rows * p.G && x.seq.row0 + qi < p.rows;
        q = (const uint16_t*)p.q + (uint64_t)(live ? x.seq.row0 + qi : 0u) * p.q_stride +
            (uint64_t)(x.h * p.G + f % p.G) * D + 16u * walk.g;
        // tokens before `limit` (a lane without a row computes another's again,
        // unmasked, and drops it)
        limit = (int32_t)(p.causal && live ? sees(x, qi) : x.seq.tokens);
    }
    // tokens that row `qi` of a causal sequence sees
    static __device__ __forceinline__ uint32_t sees(const Part& x, uint32_t qi)
    {
        const int64_t t = (int64_t)x.seq.tokens - x.seq.all + qi + 1;
        return t < 0 ? 0u : (uint32_t)t;
    }
};

template <int D>
struct Sums {
    f4_t o[D / 16];
    References ref;
    float l;
};

// What the waves note of NaN codes (take_nan), each for itself.
template <int D>
struct Noted {
    bool some[kWaves];
    uint32_t first[kWaves][D];
};

// The units of a wave's part of an item.
template <int D, int BF16, int INT8>
__device__ __forceinline__ void attend_units(const Kv8AttnParams& p, const Lane<D>& at,
                                             Sums<D>& sums, Noted<D>& noted)
{
    const uint32_t step = kWaves * kUnit, g = at.walk.g;
    const int32_t limit = at.limit;
    f4_t (&o)[D / 16] = sums.o;
    References& ref = sums.ref;
    float& l = sums.l;
    KeyBytes<D> k;
    ValueBytes<D> v;
    Entries e = at.walk.entries(at.first);
    u4_t raw[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) raw[i] = *(const u4_t*)(at.q + 64 * (i / 2) + 8 * (i & 1));
    Place now = at.walk.place(at.first, e), next;
    e = at.walk.entries(at.first + step);
    k.fetch(now.k);
    v.fetch(now.v);

    h8_t q[D / 32];
    float qf;
    {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
            const uint32_t w = raw[i / 8][(i / 2) & 3];
            most = fmaxf(most, fabsf(widen_el<BF16>((i & 1) ? w >> 16 : w & 0xffffu)));
        }
        most = fmaxf(most, xor_lanes(most, 16));
        most = fmaxf(most, xor_lanes(most, 32));
        const float shift = row_shift(most);
        qf = (1.0f / shift) * (p.scale * kLog2e);
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
            const uint32_t w = raw[i / 8][(i / 2) & 3];
            q[i / 8][i % 8] =
                (_Float16)(widen_el<BF16>((i & 1) ? w >> 16 : w & 0xffffu) * shift);
        }
    }

    // A unit. Its keys' registers are free after the scores, its values' after
    // the products: `next_keys` and `next_values` issue the next unit's loads
    // there, which then have the rest of this unit and the beginning of the next
    // to arrive.
    // `last`: the wave's last unit, the only one that rows may see parts of.
    auto take = [&](uint32_t t0, auto last, auto&& next_keys, auto&& next_values) {
        constexpr bool kLast = decltype(last)::value;
        f4_t s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    widen8<INT8>(k.x[j][i][0], k.x[j][i][1]), q[2 * i], s[j], 0, 0, 0);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    widen8<INT8>(k.x[j][i][2], k.x[j][i][3]), q[2 * i + 1], s[j], 0, 0, 0);
            }
        }
        const float fac = held_scale(now.ks) * qf, lv = __builtin_amdgcn_logf(held_scale(now.vs));
        const int live = now.live;
        __builtin_amdgcn_sched_barrier(0);
        next_keys();
        __builtin_amdgcn_sched_barrier(0);
        // the lane's tokens: strip g, token 4j + i; those it may see
        int sees = live;
        if constexpr (kLast) {
            const int ahead = limit - (int)(t0 + 16u * g);
            sees = ahead < live ? (ahead < 0 ? 0 : ahead) : live;
        }
        float most = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] *= fac;
        if (__any(sees < 16)) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[j][i] = 4 * j + i < sees ? s[j][i] : -__builtin_inff();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, s[j][i]);
        if (__any(ref.passed(most + lv, most))) {
            float product = most + lv;
            product = fmaxf(product, xor_lanes(product, 16));
            product = fmaxf(product, xor_lanes(product, 32));
            most = fmaxf(most, xor_lanes(most, 16));
            most = fmaxf(most, xor_lanes(most, 32));
            const References r = ref.moved_to(product, most);
            l *= r.s;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= r.m;
        }
        const float off = ref.exponent(lv);
        h8_t pr[2];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __builtin_amdgcn_exp2f(s[j][i] + off);
                sum += x;
                pr[j / 2][4 * (j & 1) + i] = (_Float16)x;
            }
        l += sum * ref.share(off);
        if (__any(live < 16)) {
            // a dead token's bytes may be a NaN: 0 times it is not 0
#pragma unroll
            for (int i = 0; i < D / 16; ++i) v.x[i] = live_bytes(v.x[i], live);
        }
        if constexpr (kLast && !INT8) {
            uint32_t nan = 0;
            if (__any(sees < live)) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) nan |= nan_codes(v.x[i]);
            }
            if (p.causal && threadIdx.x % 64u == 0) noted.some[threadIdx.x / 64u] = false;
            if (__any(nan)) {
                uint32_t* first = noted.first[threadIdx.x / 64u];
                for (uint32_t i = threadIdx.x % 64u; i < D; i += 64) first[i] = kNoToken;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    take_nan(v.x[i], t0 + 16u * g, &first[16 * i + at.walk.c]);
                if (threadIdx.x % 64u == 0) noted.some[threadIdx.x / 64u] = true;
            }
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<INT8>(v.x[i][0], v.x[i][1]),
                                                          pr[0], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<INT8>(v.x[i][2], v.x[i][3]),
                                                          pr[1], o[i], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        next_values();
        __builtin_amdgcn_sched_barrier(0);
    };

    uint32_t t0 = at.first;
    for (uint32_t i = 1; i < at.units; ++i, t0 += step)
        take(
            t0, Const<0>(),
            [&] {
                next = at.walk.place(t0 + step, e);
                e = at.walk.entries(t0 + 2 * step);
                k.fetch(next.k);
            },
            [&] {
                v.fetch(next.v);
                now = next;
            });
    take(t0, Const<1>(), [] {}, [] {});
    l += xor_lanes(l, 16);
    l += xor_lanes(l, 32);
}

template <int D, int BF16, int INT8>
__device__ __forceinline__ void merge_waves(const Kv8AttnParams& p, const Part& x,
                                            const Sums<D>& sums, float (*part)[kRows][D + 4],
                                            float (*stat)[kRows][3], const Noted<D>& noted)
{
    const uint32_t wave = threadIdx.x >> 6, c = threadIdx.x & 15u, g = (threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *(f4_t*)&part[wave][c][16 * i + 4 * g] = sums.o[i];
    if (g == 0) {
        stat[wave][c][0] = sums.ref.m;
        stat[wave][c][1] = sums.ref.s;
        stat[wave][c][2] = sums.l;
    }
    __syncthreads();
    const uint32_t left = x.seq.rows * p.G - x.rt * kRows;
    const uint32_t rows = left < (uint32_t)kRows ? left : kRows;
    for (uint32_t k = threadIdx.x; k < rows * (D / 4); k += kThreads) {
        const uint32_t r = k / (D / 4), ch = (k % (D / 4)) * 4;
        const uint32_t fr = x.rt * kRows + r, row = x.seq.row0 + fr / p.G;
        if (row >= p.rows) break;
        References to{stat[0][r][0], stat[0][r][1]};
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
            to = {fmaxf(to.m, stat[w][r][0]), fmaxf(to.s, stat[w][r][1])};
        f4_t a = {0, 0, 0, 0};
        float ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            ll += __builtin_amdgcn_exp2f(stat[w][r][1] - to.s) * stat[w][r][2];
            a += __builtin_amdgcn_exp2f(stat[w][r][0] - to.m) * *(const f4_t*)&part[w][r][ch];
        }
        if (!INT8 && p.causal) {
            for (int w = 0; w < kWaves; ++w) {
                if (!noted.some[w]) continue;
                const uint32_t sees = Lane<D>::sees(x, fr / p.G);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (noted.first[w][ch + i] < sees) a[i] = __builtin_nanf("");
            }
        }
        if (x.slot < 0) {
            const Quotient y(to, ll);
            const uint64_t at = (uint64_t)row * p.Hq + x.h * p.G + fr % p.G;
            *(u2_t*)((uint16_t*)p.out + at * D + ch) =
                u2_t{narrow2<BF16>(y(a[0]), y(a[1])), narrow2<BF16>(y(a[2]), y(a[3]))};
        } else {
            const uint64_t rec = (uint64_t)x.slot * p.rec_rows + r;
            *(f4_t*)(p.acc + rec * D + ch) = a;
            if (ch == 0) *(f4_t*)(p.stats + kKv8Stats * rec) = f4_t{to.m, to.s, ll, 0.0f};
        }
    }
}

template <int D, int BF16, int INT8>
__global__ __launch_bounds__(kThreads, kKv8GroupsPerCu(D)) void kv8_decode(Kv8AttnParams p,
                                                                           Divisor per_page)
{
    __shared__ float part[kWaves][kRows][D + 4];
    __shared__ float stat[kWaves][kRows][3];
    __shared__ Noted<D> noted;
    const uint32_t lane = threadIdx.x & 63u;
    Part x;
    uint32_t left = 0;  // units of the workgroup behind this part
    if (p.K) {
        const uint32_t k = blockIdx.x % p.K;
        x.b = blockIdx.x / p.K;
        x.h = blockIdx.y % p.Hkv;
        x.rt = blockIdx.y / p.Hkv;
        x.seq = Sequence(p, x.b);
        if (x.rt >= x.seq.tiles(p)) return;
        const uint32_t units = x.seq.units(), w = part_units(p, units);
        x.begin = k * w;
        if (x.begin >= units) return;
        x.end = x.begin + w < units ? x.begin + w : units;
        const uint32_t tiles = gridDim.y / p.Hkv;
        x.slot = w >= units ? -1 : (((int64_t)x.b * p.Hkv + x.h) * tiles + x.rt) * p.K + k;
    } else {
        // the quota, and the sequence that this workgroup's begins in
        uint32_t total = 0, work = 0;
        Sequence mine;
        for (uint32_t b0 = 0; b0 < p.B; b0 += 64) {
            work = 0;
            if (b0 + lane < p.B) {
                mine = Sequence(p, b0 + lane);
                work = mine.work(p);
            }
            total += __builtin_amdgcn_readlane(wave_scan(work), 63);
        }
        const uint32_t quota = quota_of(p, total);
        const uint32_t at = blockIdx.x * quota;
        if (at >= total) return;
        uint32_t before = 0;
        for (uint32_t b0 = 0;; b0 += 64) {
            if (p.B > 64) {
                work = 0;
                if (b0 + lane < p.B) {
                    mine = Sequence(p, b0 + lane);
                    work = mine.work(p);
                }
            }
            const uint32_t upto = before + wave_scan(work);
            const uint64_t past = __ballot(upto > at);
            if (past) {
                const uint32_t l = (uint32_t)__builtin_ctzll(past);
                x.b = b0 + l;
                x.seq = mine.of_lane(l);
                before = __builtin_amdgcn_readlane(upto - work, l);
                break;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
        const uint32_t units = x.seq.units(), tiles = x.seq.tiles(p);
        const uint32_t item = (at - before) / units;
        x.h = item / tiles;
        x.rt = item % tiles;
        x.begin = (at - before) % units;
        x.end = units - x.begin < quota ? units : x.begin + quota;
        x.slot = x.begin ? 2ll * blockIdx.x : x.end < units ? 2ll * blockIdx.x + 1 : -1;
        left = quota - (x.end - x.begin);
    }

    // The part behind y on the line; false at the workgroup's or the line's end.
    auto following = [&](Part& y) -> bool {
        if (left == 0) return false;
        if (++y.rt == y.seq.tiles(p)) {
            y.rt = 0;
            if (++y.h == p.Hkv) {
                y.h = 0;
                do {
                    if (++y.b >= p.B) return false;
                    y.seq = Sequence(p, y.b);
                } while (y.seq.rows == 0);
            }
        }
        const uint32_t units = y.seq.units();
        y.begin = 0;
        y.end = units < left ? units : left;
        y.slot = y.end < units ? 2ll * blockIdx.x + 1 : -1;
        left -= y.end;
        return true;
    };

    for (;;) {
        Sums<D> sums;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) sums.o[i] = f4_t{0, 0, 0, 0};
        sums.ref = References::none();
        sums.l = 0.0f;
        const Lane<D> at(p, per_page, x);
        if (at.units) attend_units<D, BF16, INT8>(p, at, sums, noted);
        else if (threadIdx.x % 64u == 0) noted.some[threadIdx.x / 64u] = false;
        merge_waves<D, BF16, INT8>(p, x, sums, part, stat, noted);
        if (!following(x)) return;
        __syncthreads();  // the merge has read its sums
    }
}

// A row's records, joined by a wave, or by TEAM of them.
template <int D, int BF16, int TEAM>
__global__ __launch_bounds__(TEAM > kWaves ? 64 * TEAM : kThreads) void kv8_combine(
    Kv8AttnParams p, uint32_t max_tiles)
{
    __shared__ float part[TEAM > 1 ? TEAM : 1][D];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    // row * Hq + head
    const uint64_t at = (uint64_t)blockIdx.x * (TEAM < kWaves ? kWaves / TEAM : 1) + wave / TEAM;
    const uint32_t row = (uint32_t)(at / p.Hq), hq = (uint32_t)(at % p.Hq);
    if (row >= p.rows) return;
    const uint32_t b = sequence_of(p, row);
    if (b >= p.B) return;
    const Sequence s(p, b);
    if (row < s.row0 || row - s.row0 >= s.rows) return;
    const uint32_t f = (row - s.row0) * p.G + hq % p.G, h = hq / p.G;
    const uint32_t rt = f / kRows, r = f % kRows;
    // its records: at most `bound` of them, the first at slot0, the others from
    // `slot` on
    uint32_t bound, apart;
    uint64_t slot0, slot;
    if (p.K) {
        bound = p.K;
        slot0 = (((uint64_t)b * p.Hkv + h) * max_tiles + rt) * p.K;
        slot = slot0 + 1;
        apart = 1;
    } else {
        uint32_t total = 0, before = 0;
        for (uint32_t b0 = 0; b0 < p.B; b0 += 64) {
            const uint32_t w = b0 + lane < p.B ? Sequence(p, b0 + lane).work(p) : 0u;
            const uint32_t upto = wave_scan(w);
            if (b - b0 < 64u) before = total + __builtin_amdgcn_readlane(upto - w, b - b0);
            total += __builtin_amdgcn_readlane(upto, 63);
        }
        const uint32_t quota = quota_of(p, total);
        const uint32_t from = before + (h * s.tiles(p) + rt) * s.units();
        const uint32_t w0 = from / quota, w1 = (from + s.units() - 1) / quota;
        bound = w1 - w0 + 1;
        slot0 = 2ull * w0 + 1;
        slot = 2ull * w0 + 2;
        apart = 2;
    }
    if (bound < 2) return;  // the whole item went to the output
    join_records<D, BF16, TEAM>(
        p, at, bound, part,
        [&](uint32_t k) {
            return (k ? slot + (uint64_t)(k - 1) * apart : slot0) * p.rec_rows + r;
        },
        [&] {
            if (p.K == 0) return bound;
            const uint32_t w = part_units(p, s.units());
            return (s.units() + w - 1) / w;
        });
}

template <int D, int BF16, int INT8>
hipError_t launch_t(hipStream_t stream, const Kv8AttnParams& p)
{
    const uint32_t tiles = (p.max_q * p.G + kRows - 1) / kRows;
    const dim3 grid = p.K ? dim3(p.B * p.K, p.Hkv * tiles) : dim3(p.groups);
    hipLaunchKernelGGL((kv8_decode<D, BF16, INT8>), grid, dim3(kThreads), 0, stream, p,
                       div_magic(p.S / 16));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.K == 1) return e;
    const uint64_t rows = (uint64_t)p.rows * p.Hq;
    const uint32_t waves = kv8_join_waves(p.K, p.groups, (uint64_t)p.B * p.Hkv * tiles);
    if (waves == 16)
        hipLaunchKernelGGL((kv8_combine<D, BF16, 16>), dim3((uint32_t)rows), dim3(1024), 0, stream,
                           p, tiles);
    else if (waves == 4)
        hipLaunchKernelGGL((kv8_combine<D, BF16, 4>), dim3((uint32_t)rows), dim3(kThreads), 0,
                           stream, p, tiles);
    else
        hipLaunchKernelGGL((kv8_combine<D, BF16, 1>), dim3((uint32_t)((rows + kWaves - 1) / kWaves)),
                           dim3(kThreads), 0, stream, p, tiles);
    return hipGetLastError();
}

template <int D>
hipError_t launch_d(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p)
{
    if (bf16) return int8 ? launch_t<D, 1, 1>(stream, p) : launch_t<D, 1, 0>(stream, p);
    return int8 ? launch_t<D, 0, 1>(stream, p) : launch_t<D, 0, 0>(stream, p);
}

}  // namespace

hipError_t launch_kv8_decode(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p)
{
    switch (p.D) {
        case 64: return launch_d<64>(stream, bf16, int8, p);
        case 128: return launch_d<128>(stream, bf16, int8, p);
        case 256: return launch_d<256>(stream, bf16, int8, p);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace tq4
