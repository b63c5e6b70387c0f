// kv8_device.hpp -- device helpers of the attention over the 8-bit paged cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_internal.hpp"
#include "tq4_device.hpp"

namespace tq4 {
namespace kv8 {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

template <int N>
struct Const {
    static constexpr int value = N;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3.0e38f;  // a running maximum before any token

// What a row's sums are held against, in log2 units and whole numbers: the products
// (weight times value scale) against 2^m, the weights against 2^s. They are two, as
// the value scales of a context may lie far apart: a page of zeros has 2^-100.
struct References {
    float m, s;

    __device__ __forceinline__ static References none() { return {kNone, kNone}; }
    // Both moved up to bring the largest product and weight to 2^6 .. 2^7, which leaves
    // the sums room until one passes 2^14; what each sum is multiplied by.
    __device__ __forceinline__ References moved_to(float product, float weight)
    {
        const References was = *this;
        m = fmaxf(m, floorf(product - 6.0f));
        s = fmaxf(s, floorf(weight - 6.0f));
        return {__builtin_amdgcn_exp2f(was.m - m), __builtin_amdgcn_exp2f(was.s - s)};
    }
    __device__ __forceinline__ bool passed(float product, float weight) const
    {
        return product > m + 14.0f || weight > s + 14.0f;
    }
    // The product of score x in a strip of value scale 2^lv is 2^(x + exponent(lv)), its
    // weight share(exponent) times that. A strip all of whose products lie below 2^-26,
    // which FP16 rounds to 0, has them at 2^-40 times its weights instead: these count
    // in their sum whatever its scale is, down to 2^-86 of the row's largest.
    __device__ __forceinline__ float exponent(float lv) const { return fmaxf(lv - m, -40.0f - s); }
    __device__ __forceinline__ float share(float exponent) const
    {
        return __builtin_amdgcn_exp2f(-(exponent + s));
    }
    // The same with less of it a tile, for strips whose lv and 2^8 / scale are at hand:
    // exponent lv - m and share rvs * gap(), once `hold` has seen the strips of a tile
    // for which `passes_or_holds`, lv the least of theirs (so a weight maybe passes). The
    // gap is at most 2^123 for scales up to 2^122. (8192 rows of 32 heads of 128 take
    // 2.9% more time with the above than with one reference, 1.3% so; the decode spills
    // with this.)
    __device__ __forceinline__ bool passes_or_holds(float product, float lv) const
    {
        return product > fminf(m, s + lv) + 14.0f || s + lv < m - 40.0f;
    }
    __device__ __forceinline__ void hold(float& lv, float& rvs) const
    {
        lv = fmaxf(lv, m - s - 40.0f);
        rvs = fminf(rvs, __builtin_amdgcn_exp2f(s - m + 48.0f));
    }
    __device__ __forceinline__ float gap() const { return __builtin_amdgcn_exp2f(m - s - 8.0f); }
};

// The sums of a row, o and l, as its output o 2^m / (l 2^s); 0 where it saw nothing.
struct Quotient {
    float inv;
    int up;

    __device__ __forceinline__ Quotient(References r, float l)
        : inv(l == 0.0f ? 0.0f : 1.0f / l),
          up((int)fminf(fmaxf(r.m - r.s, -400.0f), 400.0f))
    {
    }
    __device__ __forceinline__ float operator()(float o) const
    {
        return __builtin_amdgcn_ldexpf(o * inv, up);
    }
};

// Four codes of a word as f16 (exact for both types).
template <int INT8>
__device__ __forceinline__ void widen4(uint32_t w, h2_t& lo, h2_t& hi)
{
    if constexpr (INT8) {
        // code + 128 in the low mantissa bits of 1024: 1024 + 128 + code
        const uint32_t u = w ^ 0x80808080u;
        const h2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
        lo = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
        hi = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    } else {
        lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
}

template <int INT8>
__device__ __forceinline__ h8_t widen8(uint32_t w0, uint32_t w1)
{
    h2_t a, b, c, d;
    widen4<INT8>(w0, a, b);
    widen4<INT8>(w1, c, d);
    return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int BF16>
__device__ __forceinline__ float widen_el(uint32_t bits16)
{
    if constexpr (BF16) return __uint_as_float(bits16 << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
}

template <int BF16>
__device__ __forceinline__ uint32_t narrow2(float a, float b)
{
    if constexpr (BF16) {
        typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
        const b2_t h = {(__bf16)a, (__bf16)b};  // v_cvt_pk_bf16_f32
        return __builtin_bit_cast(uint32_t, h);
    }
    const h2_t h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
}

__device__ __forceinline__ float held_scale(float s)
{
    return fminf(fmaxf(s, kKv8LeastScale), kKv8MostScale);
}

// x scaled so that a row whose largest magnitude is `most` lies in f16's normal
// range: the power of two that brings it to [1, 2) (1 for a row of zeros).
__device__ __forceinline__ float row_shift(float most)
{
    const uint32_t e = (__float_as_uint(most) >> 23) & 0xffu;
    return e == 0u ? (most > 0.0f ? 0x1.0p+126f : 1.0f)
                   : __uint_as_float((254u - (e > 253u ? 253u : e)) << 23);
}

// n / d for n < 2^31 by the multiplier of div_magic.
struct Divisor {
    uint32_t magic, shift;
};
__device__ __forceinline__ uint32_t div_by(uint32_t n, Divisor d)
{
    return (uint32_t)(((uint64_t)n * d.magic) >> d.shift);
}
inline Divisor div_magic(uint32_t d)
{
    uint32_t shift = 31;
    while (shift < 63 && (1ull << (shift - 31)) < d) ++shift;
    return {d == 1 ? 0x80000000u : (uint32_t)((1ull << shift) / d + 1), shift};
}

// A lane's value from `CTRL`'s lane, 0 where there is none (or the row is masked).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v)
{
    return (uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v);
}

// Inclusive sum over the wave: within rows of 16 lanes by shifts, then the rows'
// last lanes to the rows behind them.
template <class T>
__device__ __forceinline__ T wave_scan(T v)
{
    v += moved<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);  // row_bcast:15 to rows 1 and 3
    v += moved<0x143, 0xc>(v);  // row_bcast:31 to rows 2 and 3
    return v;
}

// All 16 bytes of a strip's channel with those of dead tokens (>= live) zero.
__device__ __forceinline__ u4_t live_bytes(u4_t v, int live)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = live - 4 * i;
        const uint32_t m = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        v[i] &= m;
    }
    return v;
}

// NaN among the FP8 codes of values that some rows see and others do not: 0 times it
// is not 0. Such codes are taken out; the first token of each channel that had one is
// noted, and the sums of the rows that see it become NaN.
constexpr uint32_t kNoToken = ~0u;

__device__ __forceinline__ uint32_t nan_codes(uint32_t w)  // their top bits
{
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t nan_codes(u4_t w)  // not 0 where there is one
{
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) some |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;
    return some & 0x80808080u;
}
// 16 tokens of a channel, the first of them `token`.
__device__ __forceinline__ void take_nan(u4_t& w, uint32_t token, uint32_t* first)
{
    uint32_t at = kNoToken;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const uint32_t nan = (nan_codes(w[i]) >> 7) * 0xffu;
        if (nan) at = token + 4 * i + __builtin_ctz(nan) / 8;
        w[i] &= ~nan;
    }
    if (at != kNoToken) atomicMin(first, at);
}

// A sequence's rows and tokens, held in bounds.
struct SequenceBase {
    uint32_t row0, rows, all, tokens;  // rows: those computed, of all

    __device__ __forceinline__ SequenceBase() {}
    __device__ __forceinline__ SequenceBase(const Kv8AttnParams& p, uint32_t b)
    {
        row0 = b;
        all = 1;
        if (p.cu) {
            const int32_t from = p.cu[b], to = p.cu[b + 1];
            row0 = (uint32_t)from;
            all = from >= 0 && to > from ? (uint32_t)(to - from) : 0u;
        }
        rows = all < p.max_q ? all : p.max_q;
        const int32_t len = p.context_lens[b];
        const uint32_t cap = p.M * p.S;  // below 2^31
        tokens = len < 0 ? 0u : (uint32_t)len < cap ? (uint32_t)len : cap;
    }
    __device__ __forceinline__ SequenceBase of_lane(uint32_t lane) const
    {
        SequenceBase s;
        s.row0 = __builtin_amdgcn_readlane(row0, lane);
        s.rows = __builtin_amdgcn_readlane(rows, lane);
        s.all = __builtin_amdgcn_readlane(all, lane);
        s.tokens = __builtin_amdgcn_readlane(tokens, lane);
        return s;
    }
};

// The sequence that a row belongs to: the first that ends past it.
__device__ __forceinline__ uint32_t sequence_of(const Kv8AttnParams& p, uint32_t row)
{
    if (!p.cu) return row;
    uint32_t lo = 0, hi = p.B;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > (int32_t)row) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The records of output row `at`, each moved to the largest references, to the output. TEAM
// waves take them in turn and merge in `part` (TEAM rows; one wave: not used).
// record(k): the index of record k < bound; count(): how many of them were written,
// fewer than 2 where the row is none of the join's. The first loads do not wait for
// it: what they find past it is left out.
template <int D, int BF16, int TEAM, class Record, class Count>
__device__ __forceinline__ void join_records(const Kv8AttnParams& p, uint64_t at, uint32_t bound,
                                             float (*part)[D], Record&& record, Count&& count)
{
    constexpr int C = D / 64;
    const uint32_t lane = threadIdx.x & 63u, mine = (threadIdx.x >> 6) % TEAM;
    float x[8][C];
    // eight of the wave's records from k on (past the last: the last again)
    auto load = [&](uint32_t k0, uint32_t k, uint32_t last) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t kj = k0 + k + j * TEAM < last ? k0 + k + j * TEAM : last;
            __builtin_memcpy(
                x[j], __builtin_assume_aligned(p.acc + record(kj) * D + lane * C, 4 * C), 4 * C);
        }
    };
    auto stat = [&](uint32_t k) {
        return k < bound ? *(const f4_t*)(p.stats + kKv8Stats * record(k))
                         : f4_t{kNone, kNone, 0.0f, 0.0f};
    };
    f4_t st = stat(lane);
    load(0, mine, bound - 1);
    const uint32_t K = count();
    if (K < 2) return;
    References ref = References::none();
    float a[C] = {}, l = 0.0f;
    for (uint32_t k0 = 0; k0 < K; k0 += 64) {
        if (k0) {
            st = stat(k0 + lane);
            load(k0, mine, K - 1);
        }
        const bool held = k0 + lane < K;
        const References was = ref;
        if (held) ref = {fmaxf(ref.m, st[0]), fmaxf(ref.s, st[1])};
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) {
            ref.m = fmaxf(ref.m, xor_lanes(ref.m, i));
            ref.s = fmaxf(ref.s, xor_lanes(ref.s, i));
        }
        const float r = __builtin_amdgcn_exp2f(was.m - ref.m);
        const float w = held ? __builtin_amdgcn_exp2f(st[0] - ref.m) : 0.0f;  // of record k0 + lane
        l *= __builtin_amdgcn_exp2f(was.s - ref.s);
        l = held ? l + __builtin_amdgcn_exp2f(st[1] - ref.s) * st[2] : l;
#pragma unroll
        for (int i = 0; i < C; ++i) a[i] *= r;
        const uint32_t n = K - k0 < 64 ? K - k0 : 64u;
        for (uint32_t k = mine; k < n; k += 8 * TEAM) {
            if (k != mine) load(k0, k, K - 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = k + j * TEAM < n;
                const float wk = __uint_as_float(
                    __builtin_amdgcn_readlane(__float_as_uint(w), in ? k + j * TEAM : 0));
#pragma unroll
                for (int i = 0; i < C; ++i) a[i] = in ? a[i] + wk * x[j][i] : a[i];
            }
        }
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) l += xor_lanes(l, i);
    if constexpr (TEAM > 1) {
#pragma unroll
        for (int i = 0; i < C; ++i) part[mine][lane * C + i] = a[i];
        __syncthreads();
        if (mine) return;
#pragma unroll
        for (int t = 1; t < TEAM; ++t)
#pragma unroll
            for (int i = 0; i < C; ++i) a[i] += part[t][lane * C + i];
    }
    const Quotient y(ref, l);
    uint16_t* out = (uint16_t*)p.out + at * D + lane * C;
    if constexpr (C == 1) {
        *out = (uint16_t)narrow2<BF16>(y(a[0]), 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < C; i += 2) *(uint32_t*)(out + i) = narrow2<BF16>(y(a[i]), y(a[i + 1]));
    }
}

}  // namespace kv8
}  // namespace tq4
