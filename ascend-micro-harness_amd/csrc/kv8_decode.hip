// kv8_decode.hip -- attention of few rows a sequence over the 8-bit paged cache
// (tq4_kv8_paged_decode, and tq4_kv8_paged_prefill of few rows; tq4_kv8.h).
//
// Up to 16 rows (the GQA group's heads, times the query tokens) of a (sequence,
// kv head) share a pass over its tokens. A wave takes 64 tokens, four strips, at
// a time:
//   S = K Q^T     MFMA 16x16x32 f16, tokens x rows. Codes are exact in f16 and a
//                 row of q is shifted by a power of two into f16's range.
//   s' = S * (k scale * q factor) + log2(v scale)      log2 units
//   P = 2^(s' - m), in f16 with the v scale inside it, so the row's largest
//       product is 2^6 whatever the scales' spread; m moves when a row passes
//       2^14 (lazily), and the sums with it
//   O^T += V^T P^T   on V's codes;  l += P / v scale
//   out = O / l
// Tile j of S holds tokens 4j .. 4j + 3 of each of the four strips, so a lane's
// 16 scores are the 16 tokens of one strip (one scale each) for one row: they are
// the P^T operand as they lie, and the V^T operand is a channel's 16 consecutive
// bytes of that strip. Row factors are lane values; only the lazy maximum
// crosses lanes.
// Built without fast-math; the 32-bit statistics are held per wave and merged
// through LDS, then through records when a sequence is split.
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

template <int D>
struct Unit {
    u4_t k[4][D / 64];  // tile, 64 channels
    u4_t v[D / 16];     // 16 channels
    float ks, vs;
    int live;           // live tokens of the lane's strip
};

// The block-table entries behind a unit: of the strip whose keys the lane loads
// and of the strip whose values it loads; -1 past the table.
struct Entries {
    int32_t k, v;
};

template <int D, int INT8>
struct Walk {
    const Kv8AttnParams& p;
    const int32_t* table;
    Divisor per_page;   // strips of a page
    uint32_t h, L;
    uint32_t lane, c, g;

    __device__ __forceinline__ int32_t entry(uint32_t strip) const
    {
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
        return strip - div_by(strip, per_page) * (p.S / 16);
    }
    __device__ __forceinline__ void fetch(Unit<D>& u, uint32_t t0, Entries e) const
    {
        const uint32_t sk = t0 / 16 + (c >> 2), sv = t0 / 16 + g;
        const bool ok = e.v >= 0 && (uint32_t)e.v < p.P;
        const uint32_t pk = e.k >= 0 && (uint32_t)e.k < p.P ? (uint32_t)e.k : 0u;
        const uint32_t pv = ok ? (uint32_t)e.v : 0u;
        const uint64_t rk = (uint64_t)pk * p.Hkv + h, rv = (uint64_t)pv * p.Hkv + h;
        const uint8_t* k = p.key_cache + (rk * p.S + in_page(sk) * 16u + (c & 3u)) * D + 16u * g;
        const uint8_t* v = p.value_cache + (rv * p.S + in_page(sv) * 16u) * D + 16u * c;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) u.k[j][i] = *(const u4_t*)(k + 4 * j * D + 64 * i);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) u.v[i] = *(const u4_t*)(v + 256 * i);
        u.ks = p.scales[rv];
        u.vs = p.scales[(uint64_t)p.P * p.Hkv + rv];
        const int left = (int)L - (int)(16u * sv);
        u.live = !ok || left < 0 ? 0 : left > 16 ? 16 : left;
    }
};

// (seq, kv head, rows 16 rt ..) x split.
template <int D, int BF16, int INT8>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void kv8_decode(Kv8AttnParams p,
                                                                         Divisor per_page)
{
    constexpr int kPitch = D + 4;
    __shared__ float part[kWaves][kRows][kPitch];
    __shared__ float stat[kWaves][kRows][2];
    const uint32_t b = blockIdx.x / p.K, split = blockIdx.x % p.K;
    const uint32_t h = blockIdx.y % p.Hkv, rt = blockIdx.y / p.Hkv;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t c = lane & 15u, g = lane >> 4;

    // this sequence's rows and tokens
    uint32_t row0 = b, nq = 1;
    if (p.cu) {
        const int32_t a = p.cu[b], z = p.cu[b + 1];
        row0 = (uint32_t)(a < 0 ? 0 : a);
        nq = z > a && a >= 0 ? (uint32_t)(z - a) : 0u;
    }
    const uint64_t cap = (uint64_t)p.M * p.S;
    uint32_t L = p.context_lens[b] > 0 ? (uint32_t)p.context_lens[b] : 0u;
    if (L > cap) L = (uint32_t)cap;
    const uint32_t have = nq < p.max_q ? nq : p.max_q;  // rows that are computed
    if (rt * kRows >= have * p.G) return;
    const uint32_t W = split_width(L, p.kmin, p.wmin, p.wmax);
    const uint32_t begin = split * W;
    if (split > 0 && begin >= L) return;
    const uint32_t end = begin + W < L ? begin + W : L;

    // the lane's row: flat row f is token f / G, head f % G
    const uint32_t f = rt * kRows + c;
    const uint32_t qi = f / p.G, hq = h * p.G + f % p.G;
    const bool live_row = f < have * p.G && row0 + qi < p.rows;
    // tokens that it sees: before `limit`
    int64_t limit = p.causal ? (int64_t)L - nq + qi + 1 : (int64_t)L;
    if (!live_row || limit < 0) limit = 0;

    const Walk<D, INT8> walk{p, p.tables + (uint64_t)b * p.M, per_page, h, L, lane, c, g};
    const uint32_t step = kWaves * kUnit;
    const uint32_t first = begin + wave * kUnit;
    const uint32_t units = first < end ? (end - first + step - 1) / step : 0u;

    f4_t o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = f4_t{0, 0, 0, 0};
    float m = kNone, l = 0.0f;

    if (units) {
        Unit<D> ua;
        const Entries e = walk.entries(first);
        // the row of q, its channels in the order of the keys' loads
        h8_t q[D / 32];
        float qf;
        {
            float x[D / 4];
            const uint16_t* src = (const uint16_t*)p.q +
                                  (uint64_t)(live_row ? row0 + qi : 0u) * p.q_stride +
                                  (uint64_t)hq * D + 16u * g;
            u4_t raw[D / 32];
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
                raw[i] = *(const u4_t*)(src + 64 * (i / 2) + 8 * (i & 1));
            walk.fetch(ua, first, e);
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
                const uint32_t w = raw[i / 8][(i / 2) & 3];
                x[i] = live_row ? widen_el<BF16>((i & 1) ? w >> 16 : w & 0xffffu) : 0.0f;
                most = fmaxf(most, fabsf(x[i]));
            }
            most = fmaxf(most, xor_lanes(most, 16));
            most = fmaxf(most, xor_lanes(most, 32));
            const float shift = row_shift(most);
            qf = (1.0f / shift) * (p.scale * kLog2e);
#pragma unroll
            for (int i = 0; i < D / 4; ++i) q[i / 8][i % 8] = (_Float16)(x[i] * shift);
        }

        auto take = [&](const Unit<D>& u, uint32_t t0) {
            f4_t s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = f4_t{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        widen8<INT8>(u.k[j][i][0], u.k[j][i][1]), q[2 * i], s[j], 0, 0, 0);
                    s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        widen8<INT8>(u.k[j][i][2], u.k[j][i][3]), q[2 * i + 1], s[j], 0, 0, 0);
                }
            }
            const float vs = held_scale(u.vs);
            const float fac = held_scale(u.ks) * qf, lv = __builtin_amdgcn_logf(vs);
            // the lane's tokens: strip g, token 4j + i; those it may see
            const int64_t ahead = limit - (int64_t)(t0 + 16u * g);
            const int sees = ahead < u.live ? (int)(ahead < 0 ? 0 : ahead) : u.live;
            float most = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_fmaf(s[j][i], fac, lv);
                    s[j][i] = 4 * j + i < sees ? x : -__builtin_inff();
                    most = fmaxf(most, s[j][i]);
                }
            if (__any(most > m + 14.0f)) {
                most = fmaxf(most, xor_lanes(most, 16));
                most = fmaxf(most, xor_lanes(most, 32));
                const float to = fmaxf(m, most - 6.0f);
                const float r = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= r;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[i] *= r;
            }
            h8_t pr[2];
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __builtin_amdgcn_exp2f(s[j][i] - m);
                    sum += x;
                    pr[j / 2][4 * (j & 1) + i] = (_Float16)x;
                }
            l += sum * (1.0f / vs);
            const bool cut = __any(u.live < 16);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                // a dead token's bytes may be a NaN: 0 times it is not 0
                const u4_t v = cut ? live_bytes(u.v[i], u.live) : u.v[i];
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<INT8>(v[0], v[1]), pr[0],
                                                              o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen8<INT8>(v[2], v[3]), pr[1],
                                                              o[i], 0, 0, 0);
            }
        };

        for (uint32_t i = 0, t0 = first;;) {
            take(ua, t0);
            if (++i >= units) break;
            t0 += step;
            walk.fetch(ua, t0, walk.entries(t0));
        }
        l += xor_lanes(l, 16);
        l += xor_lanes(l, 32);
    }

    // merge the waves
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *(f4_t*)&part[wave][c][16 * i + 4 * g] = o[i];
    if (g == 0) {
        stat[wave][c][0] = m;
        stat[wave][c][1] = l;
    }
    __syncthreads();
    const bool whole = W >= L;  // the only split of this sequence
    const uint32_t rows = have * p.G - rt * kRows < (uint32_t)kRows ? have * p.G - rt * kRows : kRows;
    for (uint32_t k = threadIdx.x; k < rows * (D / 4); k += kThreads) {
        const uint32_t r = k / (D / 4), ch = (k % (D / 4)) * 4;
        const uint32_t fr = rt * kRows + r;
        const uint32_t row = row0 + fr / p.G;
        if (row >= p.rows) break;
        float mm = stat[0][r][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, stat[w][r][0]);
        f4_t a = {0, 0, 0, 0};
        float ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float s = __builtin_amdgcn_exp2f(stat[w][r][0] - mm);
            ll += s * stat[w][r][1];
            a += s * *(const f4_t*)&part[w][r][ch];
        }
        const uint64_t at = (uint64_t)row * p.Hq + h * p.G + fr % p.G;
        if (whole) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            *(u2_t*)((uint16_t*)p.out + at * D + ch) =
                u2_t{narrow2<BF16>(a[0] * inv, a[1] * inv), narrow2<BF16>(a[2] * inv, a[3] * inv)};
        } else {
            const uint64_t rec = at * p.K + split;
            *(f4_t*)(p.acc + rec * D + ch) = a;
            if (ch == 0) {
                p.ml[2 * rec] = mm;
                p.ml[2 * rec + 1] = ll;
            }
        }
    }
}

// The splits' records of a row, a wave each: weights 2^(m_k - max m).
template <int D, int BF16>
__global__ __launch_bounds__(kThreads) void kv8_combine(Kv8AttnParams p)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t at = (uint64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);  // row * Hq + head
    const uint32_t row = (uint32_t)(at / p.Hq);
    if (row >= p.rows) return;
    uint32_t b = row;
    if (p.cu) {
        uint32_t lo = 0, hi = p.B;  // the first sequence that ends past the row
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (p.cu[mid + 1] > (int32_t)row) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
        if (b >= p.B || p.cu[b] < 0 || p.cu[b] > (int32_t)row || row - p.cu[b] >= p.max_q) return;
    }
    const uint64_t cap = (uint64_t)p.M * p.S;
    uint32_t L = p.context_lens[b] > 0 ? (uint32_t)p.context_lens[b] : 0u;
    if (L > cap) L = (uint32_t)cap;
    const uint32_t W = split_width(L, p.kmin, p.wmin, p.wmax);
    if (W >= L) return;  // one split: written already
    const uint32_t K = (L + W - 1) / W;
    const float* ml = p.ml + 2 * at * p.K;
    float m = kNone;
    for (uint32_t k = lane; k < K; k += 64) m = fmaxf(m, ml[2 * k]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
    constexpr int C = D / 64;
    float a[C] = {}, l = 0.0f;
    const float* acc = p.acc + at * p.K * D + lane * C;
#pragma unroll 4
    for (uint32_t k = 0; k < K; ++k) {
        const float w = __builtin_amdgcn_exp2f(ml[2 * k] - m);
        l += w * ml[2 * k + 1];
        float x[C];
        __builtin_memcpy(x, __builtin_assume_aligned(acc + (uint64_t)k * D, 4 * C), 4 * C);
#pragma unroll
        for (int i = 0; i < C; ++i) a[i] += w * x[i];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* out = (uint16_t*)p.out + at * D + lane * C;
    if constexpr (C == 1) {
        *out = (uint16_t)narrow2<BF16>(a[0] * inv, 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < C; i += 2)
            *(uint32_t*)(out + i) = narrow2<BF16>(a[i] * inv, a[i + 1] * inv);
    }
}

template <int D, int BF16, int INT8>
hipError_t launch_t(hipStream_t stream, const Kv8AttnParams& p)
{
    const uint32_t tiles = (p.max_q * p.G + kRows - 1) / kRows;
    hipLaunchKernelGGL((kv8_decode<D, BF16, INT8>), dim3(p.B * p.K, p.Hkv * tiles), dim3(kThreads),
                       0, stream, p, div_magic(p.S / 16));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.K == 1) return e;
    const uint64_t rows = (uint64_t)p.rows * p.Hq;
    hipLaunchKernelGGL((kv8_combine<D, BF16>), dim3((uint32_t)((rows + kWaves - 1) / kWaves)),
                       dim3(kThreads), 0, stream, p);
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
