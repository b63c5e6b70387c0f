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
// A wave takes a (run, head, plane) whole, so nothing is shared between waves:
// the rows of a run (one, in a decode step; a page's worth in a prompt) are
// found by the wave itself from the slots around its window, and an LDS map
// from the page's offsets to rows puts any order of rows, and repeats, right.
// Keys: 16 bytes of a row a lane. Values: the lane holds its channels of all 16
// tokens of a strip, which are the strip's bytes in order, so no transpose.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_internal.hpp"
#include "tq4_device.hpp"

namespace tq4 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

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

__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
        const uint32_t o = __shfl_xor(v, s);
        v = o > v ? o : v;
    }
    return v;
}

// max over the two 16-bit magnitudes of a word, those of infinities and NaN
// left out (FIN: the largest finite magnitude's bits)
template <int BF16>
__device__ __forceinline__ uint32_t magnitude(uint32_t w, uint32_t most)
{
    constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
    if (a < inf && a > most) most = a;
    if (b < inf && b > most) most = b;
    return most;
}

// The rows of `map` (offset -> row + 1, 0: none) for plane 0: a row of D
// channels on D / 8 lanes.
template <int D, int BF16, int INT8>
__device__ __forceinline__ void write_keys(const Kv8WriteParams& p, const uint32_t* map,
                                           uint32_t page, uint32_t h, bool opened)
{
    constexpr uint32_t kLanes = D / 8, kRows = 64 / kLanes;
    const uint32_t lane = threadIdx.x & 63u, r = lane / kLanes, c = (lane % kLanes) * 8;
    const uint16_t* x = (const uint16_t*)p.key + (uint64_t)h * D + c;
    float* sp = p.scales + (uint64_t)page * p.H + h;
    const float was = *sp;
    uint32_t most = 0;
    for (uint32_t o = 0; o < p.S; o += kRows) {
        const uint32_t t = map[o + r];
        if (t) {
            const u4_t w = *(const u4_t*)(x + (uint64_t)(t - 1) * p.key_stride);
            for (int i = 0; i < 4; ++i) most = magnitude<BF16>(w[i], most);
        }
    }
    most = wave_max(most);
    const float need = needed_scale<INT8>(widen<BF16>(most));
    const float old = !opened && was > 0.0f && was < __builtin_inff() ? was : 0.0f;
    const float now = fmaxf(old, need);
    const bool move = !opened && old < now;
    const float ratio = old / now, inv = 1.0f / now;
    uint8_t* dst = p.key_cache + ((uint64_t)page * p.H + h) * p.S * D + c;
    for (uint32_t o = 0; o < p.S; o += kRows) {
        const uint32_t t = map[o + r];
        u2_t* to = (u2_t*)(dst + (uint64_t)(o + r) * D);
        if (t) {
            const u4_t w = *(const u4_t*)(x + (uint64_t)(t - 1) * p.key_stride);
            float f[8];
            for (int i = 0; i < 4; ++i) {
                f[2 * i] = widen<BF16>(w[i] & 0xffffu) * inv;
                f[2 * i + 1] = widen<BF16>(w[i] >> 16) * inv;
            }
            *to = u2_t{codes4<INT8>(f[0], f[1], f[2], f[3]), codes4<INT8>(f[4], f[5], f[6], f[7])};
        } else if (move) {
            const u2_t w = *to;
            *to = u2_t{moved4<INT8>(w[0], ratio), moved4<INT8>(w[1], ratio)};
        }
    }
    if (lane == 0) *sp = now;
}

// Plane 1: strips of 16 tokens, a lane's D / 64 channels of all of them.
template <int D, int BF16, int INT8>
__device__ __forceinline__ void write_values(const Kv8WriteParams& p, const uint32_t* map,
                                             uint32_t page, uint32_t h, bool opened)
{
    constexpr int C = D / 64;  // channels a lane
    const uint32_t lane = threadIdx.x & 63u;
    const uint16_t* x = (const uint16_t*)p.value + (uint64_t)h * D + lane * C;
    float* sp = p.scales + ((uint64_t)p.P + page) * p.H + h;
    const float was = *sp;
    auto load = [&](uint32_t t, uint32_t (&w)[(C + 1) / 2]) {
        const uint16_t* s = x + (uint64_t)(t - 1) * p.value_stride;
        if constexpr (C == 1) w[0] = *s;
        else __builtin_memcpy(w, __builtin_assume_aligned(s, 2 * C), 2 * C);
    };
    uint32_t most = 0;
    for (uint32_t o = 0; o < p.S; ++o) {
        const uint32_t t = map[o];
        if (t) {
            uint32_t w[(C + 1) / 2];
            load(t, w);
            for (int i = 0; i < (C + 1) / 2; ++i) most = magnitude<BF16>(w[i], most);
        }
    }
    most = wave_max(most);
    const float need = needed_scale<INT8>(widen<BF16>(most));
    const float old = !opened && was > 0.0f && was < __builtin_inff() ? was : 0.0f;
    const float now = fmaxf(old, need);
    const bool move = !opened && old < now;
    const float ratio = old / now, inv = 1.0f / now;
    uint8_t* dst = p.value_cache + ((uint64_t)page * p.H + h) * p.S * D + lane * C * 16;
    for (uint32_t o = 0; o < p.S; o += 16) {
        uint32_t have = 0;  // the strip's tokens that the call writes
        for (int i = 0; i < 16; ++i) have |= (map[o + i] ? 1u : 0u) << i;
        if (!have && !move) continue;
        u4_t out[C];
        if (have != 0xffffu) {
            for (int k = 0; k < C; ++k) {
                out[k] = ((const u4_t*)(dst + (uint64_t)o * D))[k];
                if (move)
                    for (int i = 0; i < 4; ++i) out[k][i] = moved4<INT8>(out[k][i], ratio);
            }
        }
        for (int i4 = 0; i4 < 4; ++i4) {  // tokens 4 * i4 .. + 3, a word a channel
            float f[C][4] = {};
            uint32_t mask = 0;
            for (int i = 0; i < 4; ++i) {
                const uint32_t t = map[o + 4 * i4 + i];
                if (t) {
                    uint32_t w[(C + 1) / 2];
                    load(t, w);
                    mask |= 0xffu << (8 * i);
                    for (int k = 0; k < C; ++k)
                        f[k][i] = widen<BF16>((w[k / 2] >> (16 * (k & 1))) & 0xffffu) * inv;
                }
            }
            for (int k = 0; k < C; ++k) {
                const uint32_t w = codes4<INT8>(f[k][0], f[k][1], f[k][2], f[k][3]);
                out[k][i4] = mask == 0xffffffffu ? w : (out[k][i4] & ~mask) | (w & mask);
            }
        }
        for (int k = 0; k < C; ++k) ((u4_t*)(dst + (uint64_t)o * D))[k] = out[k];
    }
    if (lane == 0) *sp = now;
}

// A wave per (window of `window` rows, head and plane): the runs that begin in
// the window, one after the other.
template <int D, int BF16, int INT8>
__global__ __launch_bounds__(kThreads) void kv8_writer(Kv8WriteParams p, uint32_t window)
{
    extern __shared__ uint32_t maps[];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    uint32_t* map = maps + wave * p.S;
    const uint64_t item = (uint64_t)blockIdx.x * kWaves + wave;
    const uint32_t per = 2u * p.H;
    const uint32_t first = (uint32_t)(item / per) * window;
    const uint32_t hp = (uint32_t)(item % per), h = hp >> 1;
    if (first >= p.T) return;
    const uint64_t pool = (uint64_t)p.P * p.S;
    const uint32_t last = first + window < p.T ? first + window : p.T;
    auto page_of = [&](uint32_t t) -> int64_t {
        const int32_t s = p.slots[t];
        return s >= 0 && (uint64_t)s < pool ? (int64_t)((uint32_t)s / p.S) : -1;
    };
    for (uint32_t t0 = first; t0 < last; ++t0) {
        const int64_t page = page_of(t0);
        if (page < 0 || (t0 > 0 && page_of(t0 - 1) == page)) continue;
        for (uint32_t o = lane; o < p.S; o += 64) map[o] = 0;
        wave_sync();
        for (uint32_t t = t0;; t += 64) {
            const bool in = t + lane < p.T && page_of(t + lane) == page;
            // the run goes on up to the first lane that is not in it
            const uint64_t out = ~__ballot(in);
            const uint32_t n = out ? (uint32_t)__builtin_ctzll(out) : 64u;
            if (lane < n) atomicMax(&map[(uint32_t)p.slots[t + lane] % p.S], t + lane + 1);
            if (n < 64u) break;
        }
        wave_sync();
        const bool opened = map[0] != 0;
        if (hp & 1) write_values<D, BF16, INT8>(p, map, (uint32_t)page, h, opened);
        else write_keys<D, BF16, INT8>(p, map, (uint32_t)page, h, opened);
        wave_sync();
    }
}

template <int D, int BF16, int INT8>
hipError_t launch_t(hipStream_t stream, const Kv8WriteParams& p)
{
    const uint32_t window = 1;
    const uint64_t items = (uint64_t)((p.T + window - 1) / window) * 2u * p.H;
    hipLaunchKernelGGL((kv8_writer<D, BF16, INT8>), dim3((uint32_t)((items + kWaves - 1) / kWaves)),
                       dim3(kThreads), kWaves * p.S * sizeof(uint32_t), stream, p, window);
    return hipGetLastError();
}

template <int D>
hipError_t launch_d(hipStream_t stream, int bf16, int int8, const Kv8WriteParams& p)
{
    if (bf16) return int8 ? launch_t<D, 1, 1>(stream, p) : launch_t<D, 1, 0>(stream, p);
    return int8 ? launch_t<D, 0, 1>(stream, p) : launch_t<D, 0, 0>(stream, p);
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
