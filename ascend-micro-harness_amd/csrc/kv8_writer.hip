// kv8_writer.hip -- keys and values into the 8-bit paged cache
// (tq4_kv8_reshape_and_cache, tq4_kv8.h).
//
// A run is the consecutive rows of one page. For a (run, head, plane):
//   amax over the run's finite |x|;  need = 2^e, the least with amax <= C 2^e
//   scale = max(old, need); the page's codes move to it when it grew
//   code = RN(x / scale)
// Scales are powers of two, so codes that move are shifted: an e4m3 code keeps
// its bits until it is subnormal, an INT8 code is off by at most a step in all,
// however often the scale grew (half a step each time, of a step that doubles).
//
// Runs of several rows (prompts) go to waves a strip of 16 offsets each, up to
// eight waves a page, which exchange their amax; an LDS map from the page's offsets
// to rows puts any order of rows, and repeats, right. Single rows (a decode step)
// go to 16 lanes each. Waves find their runs themselves, from the slots of a window
// of rows and its neighbours.
//
// Memory bounds the prompts: 16384 rows of 8 heads of 128 24.3 us, 4.1 TB/s of the
// 4.9 that a copy reaches (a wave a whole page: 34 us, its strips one after the
// other). 64 single rows 3.8 us, a launch; a wave a row instead of 16 lanes 6.0. Pages
// whose scale grows are moved one after the other by the wave that wrote their row: where
// all 512 (page, head) pairs of 64 rows grow, 5 / 22 / 45 us more in pages of 16 / 64 / 128.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_internal.hpp"
#include "tq4_device.hpp"

namespace tq4 {
namespace {

// waves of a workgroup: four, or a team's
constexpr int waves_of(int team) { return team > 4 ? team : 4; }

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

// Orders a wave's LDS accesses for the compiler (the hardware keeps them in order).
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int BF16>
__device__ __forceinline__ float widen(uint32_t bits16)
{
    if constexpr (BF16) return __uint_as_float(bits16 << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
}

// Four values (already divided by the scale) as four codes.
template <int INT8>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d)
{
    constexpr float M = INT8 ? 127.0f : 448.0f;
    // min first: a NaN becomes +M
    a = fmaxf(fminf(a, M), -M);
    b = fmaxf(fminf(b, M), -M);
    c = fmaxf(fminf(c, M), -M);
    d = fmaxf(fminf(d, M), -M);
    if constexpr (INT8) {
        // 1.5 * 2^23 + x: the sum's rounding is x's to nearest even, the code
        // its low byte
        const uint32_t ia = __float_as_uint(a + 12582912.0f), ib = __float_as_uint(b + 12582912.0f);
        const uint32_t ic = __float_as_uint(c + 12582912.0f), id = __float_as_uint(d + 12582912.0f);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(id, ic, 0x0c0c0400),
                                     __builtin_amdgcn_perm(ib, ia, 0x0c0c0400), 0x05040100);
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
        return (uint32_t)w;
    }
}

// The four codes of a word times `ratio` (at most 1), rounded again.
template <int INT8>
__device__ __forceinline__ uint32_t moved4(uint32_t w, float ratio)
{
    if constexpr (INT8) {
        const float a = (float)(int8_t)w, b = (float)(int8_t)(w >> 8);
        const float c = (float)(int8_t)(w >> 16), d = (float)(int8_t)(w >> 24);
        return codes4<1>(a * ratio, b * ratio, c * ratio, d * ratio);
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * ratio, lo[1] * ratio, 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * ratio, hi[1] * ratio, r, true);
        // a NaN code (from another writer) keeps its byte, sign and all
        const uint32_t nan = ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
        return ((uint32_t)r & ~nan) | (w & nan);
    }
}

// The least power of two s >= 2^-100 with amax <= C s. C is 1.75 * 2^8 or
// (127/64) * 2^6: the exponent is amax's less 8 (6), one more when amax's
// fraction lies above C's.
template <int INT8>
__device__ __forceinline__ float needed_scale(float amax)
{
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - (INT8 ? 6 : 8) + ((u & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u));
    const float s = __uint_as_float((uint32_t)(e < 27 ? 27 : e) << 23);  // 27: 2^-100
    return s;
}

// The largest of all lanes' values.
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t o = __float_as_uint(xor_lanes(__uint_as_float(v), s));
        v = o > v ? o : v;
    }
    return v;
}

typedef uint16_t us2_t __attribute__((ext_vector_type(2)));

// Magnitudes of two elements' bits, the larger of each half kept.
__device__ __forceinline__ us2_t larger(us2_t most, uint32_t w)
{
    return __builtin_elementwise_max(most, __builtin_bit_cast(us2_t, w & 0x7fff7fffu));
}

// The same without infinities and NaN.
template <int BF16>
__device__ __forceinline__ us2_t larger_finite(us2_t most, uint32_t w)
{
    constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
    if ((w & 0x7fffu) >= inf) w &= 0xffff0000u;
    if (((w >> 16) & 0x7fffu) >= inf) w &= 0x0000ffffu;
    return larger(most, w);
}

// What a (run, head, plane) does to its page.
struct Scale {
    float now, inv, ratio;
    bool move;
};
template <int BF16, int INT8>
__device__ __forceinline__ Scale next_scale(float was, uint32_t amax_bits, bool opened)
{
    const float need = needed_scale<INT8>(widen<BF16>(amax_bits));
    const float old = !opened && was > 0.0f && was < __builtin_inff() ? was : 0.0f;
    Scale s;
    s.now = fmaxf(old, need);
    s.move = !opened && old < s.now;
    s.ratio = old / s.now;
    s.inv = 1.0f / s.now;
    return s;
}

// A run's rows: map[offset in the page] = row + 1, or 0. `any` is a row of the
// run, which stands in where a load needs an address.
struct Run {
    const uint32_t* map;
    uint32_t any, page, strips;
    bool opened;
};

// The waves that share a page: wave `at` of TEAM takes strips at, at + TEAM, ..
// of it. lds: two words a wave of the workgroup, whose teams all make the same calls.
template <int TEAM>
struct Team {
    uint32_t at;
    uint32_t (*lds)[2];

    __device__ __forceinline__ void max(uint32_t& a, uint32_t& b) const
    {
        if constexpr (TEAM > 1) {
            const uint32_t wave = threadIdx.x >> 6;
            __syncthreads();  // the last call's reads
            if ((threadIdx.x & 63u) == 0) {
                lds[wave][0] = a;
                lds[wave][1] = b;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TEAM; ++i) {
                const uint32_t x = lds[wave - at + i][0], y = lds[wave - at + i][1];
                a = x > a ? x : a;
                b = y > b ? y : b;
            }
        }
    }
};

// The amax of what `each(f)` feeds to f.
template <int BF16, class Each>
__device__ __forceinline__ uint32_t amax_bits(Each&& each)
{
    constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
    us2_t m = {0, 0};
    each([&](uint32_t w) { m = larger(m, w); });
    uint32_t most = wave_max(m[0] > m[1] ? m[0] : m[1]);
    if (most >= inf) {
        m = us2_t{0, 0};
        each([&](uint32_t w) { m = larger_finite<BF16>(m, w); });
        most = wave_max(m[0] > m[1] ? m[0] : m[1]);
    }
    return most;
}

// Keys of a run: a row of D channels lies on D / 8 lanes, a strip of 16 rows in
// D / 32 loads.
template <int D, int BF16, int INT8>
struct Keys {
    static constexpr uint32_t kLanes = D / 8, kRows = 64 / kLanes;
    static constexpr int kPasses = 16 / kRows;
    struct Strip {
        u4_t w[kPasses];
        uint32_t have;  // passes in which the lane's row is written
    };
    const uint16_t* x;
    uint64_t stride;
    uint8_t* dst;
    const uint32_t* map;
    uint32_t any, r;

    __device__ __forceinline__ Keys(const Kv8WriteParams& p, const Run& run, uint32_t h)
    {
        const uint32_t lane = threadIdx.x & 63u, c = (lane % kLanes) * 8;
        r = lane / kLanes;
        x = (const uint16_t*)p.key + (uint64_t)h * D + c;
        stride = p.key_stride;
        dst = p.key_cache + (((uint64_t)run.page * p.H + h) * p.S + r) * D + c;
        map = run.map;
        any = run.any;
    }
    __device__ __forceinline__ void load(Strip& s, uint32_t j) const
    {
        s.have = 0;
#pragma unroll
        for (int q = 0; q < kPasses; ++q) {
            const uint32_t t = map[16 * j + q * kRows + r];
            s.have |= (t ? 1u : 0u) << q;
            s.w[q] = *(const u4_t*)(x + (uint64_t)(t ? t - 1 : any) * stride);
        }
    }
    template <class F>
    __device__ __forceinline__ void feed(const Strip& s, F& f) const
    {
#pragma unroll
        for (int q = 0; q < kPasses; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) f((s.have >> q) & 1u ? s.w[q][i] : 0u);
    }
    __device__ __forceinline__ void store(const Strip& s, uint32_t j, const Scale& sc) const
    {
        u2_t held[kPasses];
        if (sc.move) {
#pragma unroll
            for (int q = 0; q < kPasses; ++q)
                held[q] = *(const u2_t*)(dst + (uint64_t)(16 * j + q * kRows) * D);
        }
#pragma unroll
        for (int q = 0; q < kPasses; ++q) {
            u2_t* to = (u2_t*)(dst + (uint64_t)(16 * j + q * kRows) * D);
            if ((s.have >> q) & 1u) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f[2 * i] = widen<BF16>(s.w[q][i] & 0xffffu) * sc.inv;
                    f[2 * i + 1] = widen<BF16>(s.w[q][i] >> 16) * sc.inv;
                }
                *to = u2_t{codes4<INT8>(f[0], f[1], f[2], f[3]),
                           codes4<INT8>(f[4], f[5], f[6], f[7])};
            } else if (sc.move) {
                *to = u2_t{moved4<INT8>(held[q][0], sc.ratio), moved4<INT8>(held[q][1], sc.ratio)};
            }
        }
    }
};

// Values of a run: the lane holds its D / 64 channels of a strip's 16 tokens,
// which are 16 consecutive bytes a channel. A strip that the run covers in part
// is read and written back whole.
template <int D, int BF16, int INT8>
struct Values {
    static constexpr int C = D / 64;  // channels a lane
    static constexpr int kWords = (C + 1) / 2;
    struct Strip {
        uint32_t w[16][kWords];
        uint32_t have;  // tokens that are written (the same in every lane)
    };
    const uint16_t* x;
    uint64_t stride;
    uint8_t* dst;
    const uint32_t* map;
    uint32_t any;

    __device__ __forceinline__ Values(const Kv8WriteParams& p, const Run& run, uint32_t h)
    {
        const uint32_t lane = threadIdx.x & 63u;
        x = (const uint16_t*)p.value + (uint64_t)h * D + lane * C;
        stride = p.value_stride;
        dst = p.value_cache + ((uint64_t)run.page * p.H + h) * p.S * D + lane * C * 16;
        map = run.map;
        any = run.any;
    }
    __device__ __forceinline__ void load(Strip& s, uint32_t j) const
    {
        s.have = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t t = __builtin_amdgcn_readfirstlane(map[16 * j + i]);
            s.have |= (t ? 1u : 0u) << i;
            const uint16_t* src = x + (uint64_t)(t ? t - 1 : any) * stride;
            if constexpr (C == 1) s.w[i][0] = *src;
            else __builtin_memcpy(s.w[i], __builtin_assume_aligned(src, 2 * C), 2 * C);
        }
    }
    template <class F>
    __device__ __forceinline__ void feed(const Strip& s, F& f) const
    {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((s.have >> i) & 1u) {
#pragma unroll
                for (int k = 0; k < kWords; ++k) f(s.w[i][k]);
            }
    }
    __device__ __forceinline__ void store(const Strip& s, uint32_t j, const Scale& sc) const
    {
        if (!s.have && !sc.move) return;
        u4_t* to = (u4_t*)(dst + (uint64_t)j * 16 * D);
        u4_t held[C];
        if (s.have != 0xffffu) {
#pragma unroll
            for (int k = 0; k < C; ++k) held[k] = to[k];
            if (sc.move) {
#pragma unroll
                for (int k = 0; k < C; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) held[k][i] = moved4<INT8>(held[k][i], sc.ratio);
            }
        }
#pragma unroll
        for (int k = 0; k < C; ++k) {
            u4_t out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f[4];
                uint32_t mask = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[e] = widen<BF16>((s.w[4 * i + e][k / 2] >> (16 * (k & 1))) & 0xffffu) * sc.inv;
                    mask |= ((s.have >> (4 * i + e)) & 1u) * (0xffu << (8 * e));
                }
                const uint32_t w = codes4<INT8>(f[0], f[1], f[2], f[3]);
                out[i] = s.have == 0xffffu ? w : (held[k][i] & ~mask) | (w & mask);
            }
            to[k] = out;
        }
    }
};

// Both planes of a (run, head). The wave's first strip stays in registers between
// the amax and the codes; the others of a larger page are read again.
template <int D, int BF16, int INT8, int TEAM>
__device__ __forceinline__ void write_page(const Kv8WriteParams& p, const Run& run, uint32_t h,
                                           const Team<TEAM>& team)
{
    typedef Keys<D, BF16, INT8> K;
    typedef Values<D, BF16, INT8> V;
    const K keys(p, run, h);
    const V values(p, run, h);
    float* sk = p.scales + (uint64_t)run.page * p.H + h;
    float* sv = sk + (uint64_t)p.P * p.H;
    typename K::Strip k;
    typename V::Strip v;
    const bool some = team.at < run.strips;
    if (some) {
        keys.load(k, team.at);
        values.load(v, team.at);
    }
    const float was_k = *sk, was_v = *sv;
    auto most = [&](auto& x, auto& kept) {
        return amax_bits<BF16>([&](auto&& f) {
            if (some) x.feed(kept, f);
            for (uint32_t j = team.at + TEAM; j < run.strips; j += TEAM) {
                auto s = kept;
                x.load(s, j);
                x.feed(s, f);
            }
        });
    };
    uint32_t mk = most(keys, k), mv = most(values, v);
    team.max(mk, mv);
    const Scale a = next_scale<BF16, INT8>(was_k, mk, run.opened);
    const Scale b = next_scale<BF16, INT8>(was_v, mv, run.opened);
    auto store = [&](auto& x, auto& kept, const Scale& sc) {
        if (some) x.store(kept, team.at, sc);
        for (uint32_t j = team.at + TEAM; j < run.strips; j += TEAM) {
            auto s = kept;
            x.load(s, j);
            x.store(s, j, sc);
        }
    };
    store(keys, k, a);
    store(values, v, b);
    if ((threadIdx.x & 63u) == 0 && team.at == 0) {
        *sk = a.now;
        *sv = b.now;
    }
}

// A row whose run is the row alone (a decode step's) takes 16 lanes of a wave for
// both planes of a head: the codes go straight to their places, a byte a channel
// in the values' strip. Where the page's scale grew, the whole wave moves the page.

// Plane 0 of a page, but its offset `at`, to a scale that grew.
template <int D, int INT8>
__device__ __forceinline__ void move_keys(const Kv8WriteParams& p, uint64_t row0, uint32_t at,
                                          float ratio)
{
    constexpr uint32_t kLanes = D / 8, kRows = 64 / kLanes;
    const uint32_t lane = threadIdx.x & 63u, r = lane / kLanes;
    uint8_t* dst = p.key_cache + (row0 * p.S + r) * D + (lane % kLanes) * 8;
    for (uint32_t o = 0; o < p.S; o += 16) {
        u2_t w[16 / kRows];
#pragma unroll
        for (uint32_t q = 0; q < 16 / kRows; ++q)
            w[q] = *(const u2_t*)(dst + (uint64_t)(o + q * kRows) * D);
#pragma unroll
        for (uint32_t q = 0; q < 16 / kRows; ++q)
            if (o + q * kRows + r != at)
                *(u2_t*)(dst + (uint64_t)(o + q * kRows) * D) =
                    u2_t{moved4<INT8>(w[q][0], ratio), moved4<INT8>(w[q][1], ratio)};
    }
}

// Plane 1 of a page to a scale that grew; the codes of its offset `at` are `fresh`.
template <int D, int INT8>
__device__ __forceinline__ void move_values(const Kv8WriteParams& p, uint64_t row0, uint32_t at,
                                            float ratio, const uint8_t* fresh)
{
    constexpr int C = D / 64;
    const uint32_t lane = threadIdx.x & 63u;
    uint8_t* dst = p.value_cache + row0 * p.S * D + lane * C * 16;
    for (uint32_t o = 0; o < p.S; o += 16) {
        u4_t* to = (u4_t*)(dst + (uint64_t)o * D);
#pragma unroll
        for (int k = 0; k < C; ++k) {
            u4_t w = to[k];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = moved4<INT8>(w[i], ratio);
                if (at / 4 == o / 4 + i) {
                    const uint32_t sh = 8 * (at % 4);
                    w[i] = (w[i] & ~(0xffu << sh)) | (uint32_t)fresh[lane * C + k] << sh;
                }
            }
            to[k] = w;
        }
    }
}

// The largest magnitude over the 16 lanes of a row, of N words a lane.
template <int BF16, int N>
__device__ __forceinline__ uint32_t row_amax(const uint32_t (&w)[N])
{
    auto over = [&](us2_t m) {
        uint32_t v = m[0] > m[1] ? m[0] : m[1];
#pragma unroll
        for (int s = 1; s < 16; s <<= 1) {
            const uint32_t o = __float_as_uint(xor_lanes(__uint_as_float(v), s));
            v = o > v ? o : v;
        }
        return v;
    };
    us2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) m = larger(m, w[i]);
    uint32_t v = over(m);
    if (__any(v >= (BF16 ? 0x7f80u : 0x7c00u))) {
        m = us2_t{0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) m = larger_finite<BF16>(m, w[i]);
        v = over(m);
    }
    return v;
}

constexpr uint32_t kMostRows = 62;  // of a window: a wave sees the rows beside it too

// The window that a wave works on: lane i sees row first - 1 + i.
struct Window {
    uint32_t first, rows;
    uint32_t page;  // the lane's row's, or ~0

    __device__ __forceinline__ Window(const Kv8WriteParams& p, uint32_t first_, uint32_t rows_)
        : first(first_), rows(rows_)
    {
        page = page_at(p, first - 1 + (threadIdx.x & 63u));  // (first 0: lane 0 reads nothing)
    }
    static __device__ __forceinline__ uint32_t page_at(const Kv8WriteParams& p, uint32_t t)
    {
        const uint32_t s = t < p.T ? (uint32_t)p.slots[t] : ~0u;
        return s < p.P * p.S ? s / p.S : ~0u;  // at most 2^31 slots
    }
    // the lanes whose rows begin a run, and those whose runs go on behind them
    __device__ __forceinline__ uint64_t leaders() const
    {
        const uint32_t lane = threadIdx.x & 63u, before = __shfl_up(page, 1);
        return __ballot(lane >= 1 && lane <= rows && page != ~0u && page != before);
    }
    __device__ __forceinline__ uint64_t longer() const
    {
        return __ballot(page == __shfl_down(page, 1));
    }
};

// A workgroup's single rows, a (row, head) to 16 lanes.
template <int D, int BF16, int INT8, int kWaves>
__device__ __forceinline__ void write_single_rows(const Kv8WriteParams& p, uint32_t first,
                                                  uint32_t rows, uint32_t* lds)
{
    constexpr int N = D / 32;       // words of elements a lane: D / 16 channels
    constexpr int kBytes = D / 16;  // codes a lane
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u, l = lane & 15u;
    const Window win(p, first, rows);
    const uint64_t single = win.leaders() & ~win.longer();
    if (!single) return;
    // the wave's own list of them
    uint32_t* list = lds + wave * 64;
    uint8_t* stage = (uint8_t*)(lds + kWaves * 64) + wave * 4 * D;
    if ((single >> lane) & 1u) list[__builtin_popcountll(single & ((1ull << lane) - 1))] = lane;
    wave_sync();
    const uint32_t pairs = (uint32_t)__builtin_popcountll(single) * p.H;
    for (uint32_t i0 = wave * 4; i0 < pairs; i0 += kWaves * 4) {
        const uint32_t i = i0 + lane / 16;
        const bool on = i < pairs;
        const uint32_t at = list[on ? i / p.H : 0], h = on ? i % p.H : 0;
        const uint32_t t = first - 1 + at;
        const uint32_t slot = (uint32_t)p.slots[t], page = slot / p.S, off = slot - page * p.S;
        uint32_t k[N], v[N];
        const uint64_t x = (uint64_t)h * D + l * (D / 16);
        const void* ks = (const uint16_t*)p.key + t * p.key_stride + x;
        const void* vs = (const uint16_t*)p.value + t * p.value_stride + x;
        __builtin_memcpy(k, __builtin_assume_aligned(ks, D / 8 < 16 ? D / 8 : 16), D / 8);
        __builtin_memcpy(v, __builtin_assume_aligned(vs, D / 8 < 16 ? D / 8 : 16), D / 8);
        const uint64_t row0 = (uint64_t)page * p.H + h;
        float* sk = p.scales + row0;
        float* sv = sk + (uint64_t)p.P * p.H;
        const float was_k = *sk, was_v = *sv;
        const Scale a = next_scale<BF16, INT8>(was_k, row_amax<BF16>(k), off == 0);
        const Scale b = next_scale<BF16, INT8>(was_v, row_amax<BF16>(v), off == 0);
        uint32_t ck[(kBytes + 3) / 4], cv[(kBytes + 3) / 4];
        auto codes = [](const uint32_t (&w)[N], float inv, uint32_t (&c)[(kBytes + 3) / 4]) {
#pragma unroll
            for (int j = 0; j < kBytes / 4; ++j)
                c[j] = codes4<INT8>(widen<BF16>(w[2 * j] & 0xffffu) * inv,
                                    widen<BF16>(w[2 * j] >> 16) * inv,
                                    widen<BF16>(w[2 * j + 1] & 0xffffu) * inv,
                                    widen<BF16>(w[2 * j + 1] >> 16) * inv);
        };
        codes(k, a.inv, ck);
        codes(v, b.inv, cv);
        // the values' codes change lanes: lane l then holds channels l, l + 16, ..
        uint8_t* mine = stage + lane / 16 * D;
        wave_sync();
        __builtin_memcpy(__builtin_assume_aligned(mine + l * kBytes, 4), cv, kBytes);
        wave_sync();
        uint64_t moves = __ballot(on && a.move && l == 0);
        while (moves) {
            const int src = __builtin_ctzll(moves);
            moves &= moves - 1;
            const uint64_t r0 = (uint64_t)__builtin_amdgcn_readlane(page, src) * p.H +
                                __builtin_amdgcn_readlane(h, src);
            move_keys<D, INT8>(p, r0, __builtin_amdgcn_readlane(off, src),
                               __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(a.ratio), src)));
        }
        moves = __ballot(on && b.move && l == 0);
        while (moves) {
            const int src = __builtin_ctzll(moves);
            moves &= moves - 1;
            const uint64_t r0 = (uint64_t)__builtin_amdgcn_readlane(page, src) * p.H +
                                __builtin_amdgcn_readlane(h, src);
            move_values<D, INT8>(p, r0, __builtin_amdgcn_readlane(off, src),
                                 __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(b.ratio), src)),
                                 stage + src / 16 * D);
        }
        if (on) {
            __builtin_memcpy(__builtin_assume_aligned(p.key_cache + (row0 * p.S + off) * D + l * kBytes, 4),
                             ck, kBytes);
            if (!b.move) {
                uint8_t* to = p.value_cache + row0 * p.S * D + off / 16 * 16 * D + off % 16 + 16 * l;
#pragma unroll
                for (int j = 0; j < kBytes; ++j) to[256 * j] = mine[16 * j + l];
            }
            if (l == 0) {
                *sk = a.now;
                *sv = b.now;
            }
        }
    }
}

// The runs of several rows that begin in a window, one after the other, a team of
// waves a head, `each` of them in turn.
template <int D, int BF16, int INT8, int TEAM>
__device__ __forceinline__ void write_runs(const Kv8WriteParams& p, uint32_t block, uint32_t rows,
                                           uint32_t each, uint32_t* lds)
{
    constexpr uint32_t kWaves = waves_of(TEAM), kItems = kWaves / TEAM;
    __shared__ uint32_t shared[kWaves][2];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    uint32_t* map = lds + wave * p.S;
    const Team<TEAM> team{wave % TEAM, shared};
    // The items of a workgroup have one window, so its teams meet at the same
    // barriers: its heads are padded to whole workgroups.
    const uint32_t per = (p.H + kItems * each - 1) / (kItems * each);
    const uint32_t first = block / per * rows;
    if (first >= p.T) return;
    const Window win(p, first, rows);
    uint64_t leaders = win.leaders() & win.longer();
    while (leaders) {
        const uint32_t at = (uint32_t)__builtin_ctzll(leaders);  // lane of the run's first row
        leaders &= leaders - 1;
        const uint32_t t0 = first - 1 + at;
        const uint32_t page = __builtin_amdgcn_readlane(win.page, at);
        wave_sync();
        for (uint32_t o = lane; o < p.S; o += 64) map[o] = 0;
        wave_sync();
        // the rows from t0 on, up to the first of another page; the later row of
        // a slot stays
        uint64_t out = ~__ballot(win.page == page) >> at;
        uint32_t n = out ? (uint32_t)__builtin_ctzll(out) : 64u - at;
        if (lane >= at && lane < at + n)
            atomicMax(&map[(uint32_t)p.slots[t0 + (lane - at)] - page * p.S], t0 + (lane - at) + 1);
        if (n == 64u - at) {
            for (uint32_t t = first + 63;; t += 64) {
                out = ~__ballot(Window::page_at(p, t + lane) == page);
                n = out ? (uint32_t)__builtin_ctzll(out) : 64u;
                if (lane < n) atomicMax(&map[(uint32_t)p.slots[t + lane] - page * p.S], t + lane + 1);
                if (n < 64u) break;
            }
        }
        wave_sync();
        Run run;
        run.map = map;
        run.any = t0;
        run.page = page;
        run.strips = p.S / 16;
        run.opened = __builtin_amdgcn_readfirstlane(map[0]) != 0;
        for (uint32_t e = 0; e < each; ++e) {
            const uint32_t h = __builtin_amdgcn_readfirstlane(((block % per) * each + e) * kItems +
                                                              wave / TEAM);
            if (h < p.H) {
                write_page<D, BF16, INT8, TEAM>(p, run, h, team);
            } else {  // a head too many: the barriers alone
                uint32_t x = 0, y = 0;
                team.max(x, y);
            }
        }
    }
}

// Workgroups below `blocks` take the single rows of `rows` rows each, the others
// runs.
struct Deal {
    uint32_t blocks, rows;            // single rows
    uint32_t window, each;            // runs
};

template <int D, int BF16, int INT8, int TEAM>
__global__ __launch_bounds__(64 * waves_of(TEAM), D < 256 ? 4 : 3) void kv8_writer(
    Kv8WriteParams p, Deal deal)
{
    extern __shared__ uint32_t lds[];
    if (blockIdx.x < deal.blocks)
        write_single_rows<D, BF16, INT8, waves_of(TEAM)>(p, blockIdx.x * deal.rows, deal.rows, lds);
    else
        write_runs<D, BF16, INT8, TEAM>(p, blockIdx.x - deal.blocks, deal.window, deal.each,
                                            lds);
}

template <int D, int BF16, int INT8, int TEAM>
hipError_t launch_t(hipStream_t stream, const Kv8WriteParams& p)
{
    constexpr uint32_t kWaves = waves_of(TEAM), kItems = kWaves / TEAM;
    Deal deal;
    // A workgroup costs about 4 ns of the launch whether it finds work or not:
    // at most 512 for the single rows, with 16 (row, head) pairs at least, and
    // about two thousand for the runs, whose windows are a page of rows or as much
    // of one as a wave sees; where that leaves CUs idle, less of it, and fewer runs
    // one after the other (2900 rows of 4 heads of 64 in pages of 32: 9.8 us with
    // windows of 32 rows, 7.2 of 16).
    deal.rows = (p.T + 511) / 512;
    if (deal.rows * p.H < 16) deal.rows = (15 + p.H) / p.H;
    if (deal.rows > kMostRows) deal.rows = kMostRows;
    deal.blocks = (p.T + deal.rows - 1) / deal.rows;
    deal.window = p.S < kMostRows ? p.S : kMostRows;
    const uint64_t items = ((uint64_t)p.H + kItems - 1) / kItems;
    while (deal.window > 8 && (p.T / deal.window + 1) * items < 512)
        deal.window = deal.window > 32 ? 32 : deal.window / 2;
    const uint64_t windows = (p.T + deal.window - 1) / deal.window;
    uint64_t each = windows * items / 2048;
    if (each > items) each = items;
    if (each < 1) each = 1;
    deal.each = (uint32_t)each;
    const uint64_t per = (p.H + kItems * each - 1) / (kItems * each);
    const size_t maps = kWaves * p.S * sizeof(uint32_t);
    const size_t lists = kWaves * (64 * sizeof(uint32_t) + 4 * D);
    hipLaunchKernelGGL((kv8_writer<D, BF16, INT8, TEAM>),
                       dim3((uint32_t)(deal.blocks + windows * per)), dim3(64 * kWaves),
                       maps > lists ? maps : lists, stream, p, deal);
    return hipGetLastError();
}

// A wave a strip of the page, up to eight.
template <int D, int BF16, int INT8>
hipError_t launch_s(hipStream_t stream, const Kv8WriteParams& p)
{
    if (p.S <= 16) return launch_t<D, BF16, INT8, 1>(stream, p);
    if (p.S <= 32) return launch_t<D, BF16, INT8, 2>(stream, p);
    if (p.S <= 64) return launch_t<D, BF16, INT8, 4>(stream, p);
    return launch_t<D, BF16, INT8, 8>(stream, p);
}

template <int D>
hipError_t launch_d(hipStream_t stream, int bf16, int int8, const Kv8WriteParams& p)
{
    if (bf16) return int8 ? launch_s<D, 1, 1>(stream, p) : launch_s<D, 1, 0>(stream, p);
    return int8 ? launch_s<D, 0, 1>(stream, p) : launch_s<D, 0, 0>(stream, p);
}

}  // namespace

hipError_t launch_kv8_writer(hipStream_t stream, int bf16, int int8, const Kv8WriteParams& p)
{
    switch (p.D) {
        case 64: return launch_d<64>(stream, bf16, int8, p);
        case 128: return launch_d<128>(stream, bf16, int8, p);
        case 256: return launch_d<256>(stream, bf16, int8, p);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace tq4
