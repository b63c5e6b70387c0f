// kv8_prefill.hip -- attention of many rows a sequence over the 8-bit paged cache
// (tq4_kv8_paged_prefill of prompt chunks and cross attention; tq4_kv8.h).
//
// A workgroup takes 128 or 256 rows of a (sequence, kv head): query tokens times
// the GQA group's heads, so the group shares each key. A wave has 32 of them and
// walks the tokens 64 at a time with its workgroup:
//   S = K Q^T       MFMA 32x32x16 f16, 32 tokens x 32 rows
//   s' = S * (k scale * q factor)
//   P = 2^(s' + log2(v scale) - m)  in f16, the v scale inside it (kv8_decode.hip)
//   O^T += V^T P^T, l += 2^(s' - s), out = O 2^m / (l 2^s)
// The tile's codes are widened to f16 once, on their way into LDS, in the order in
// which the matrix operands are read (a lane's 16 bytes next to its neighbour's).
// Tokens are permuted inside a block of 32 so that a lane's scores are, as they
// lie, the P^T operand of 8 consecutive tokens of a strip, half a value row: row
// m = 16 s + 8 a + 4 half + i of the block is token 16 s + 8 half + 4 a + i.
// Two LDS buffers: tile j is computed while tile j + 1 is widened into the other
// and tile j + 2 comes from memory.
//
// Arithmetic bounds it: 8192 causal rows of 32 heads of 128 (8 KV heads) 556 us, 988
// TFLOP/s where a library product of f16 matrices reaches 1284 to 1336; of 32 heads of
// 64 355 us, 775; of 16 heads of 256 808 us, 681 (its 32 rows fill a wave's registers:
// one wave a SIMD). (Cards and their clocks differ by up to 12%.) An earlier form, of
// 616 us, took 426 without the softmax and the widening, which added about 100 each; a
// ring of operand blocks and table entries that nothing waits for made up the
// difference. Issue order otherwise
// is not what holds it: priorities for one of a SIMD's two waves, a wave half a tile
// behind the other, and a tile's softmax beside the next one's scores in one wave all
// took as long or longer. 64 rows a wave halve the LDS reads, but their sums move
// through the accumulation registers, which cost more.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8_device.hpp"

namespace tq4 {
namespace {

using namespace kv8;

typedef float f16_t __attribute__((ext_vector_type(16)));

constexpr int kTile = 64;             // tokens
constexpr int kStrips = kTile / 16;

// Rows of a workgroup of W waves.
constexpr uint32_t group_rows(int w) { return 32u * w; }

// LDS of a tile: operand blocks of 64 lanes x 16 bytes. Keys: [block of 32
// tokens][16 channels]; values: [strip][32 channels]. Key blocks lie 16 bytes
// further apart than their size, which spreads a wave's stores over the banks.
template <int D>
struct Tile {
    static constexpr int kKeyBlock = 1024 + 16;
    static constexpr int kKeys = 2 * (D / 16) * kKeyBlock;
    static constexpr int kValues = kStrips * (D / 32) * 1024;
    static constexpr int kBytes = kKeys + kValues;
};

struct StripInfo {
    float ks, lv, rvs;  // key scale, log2 of the value scale, 2^8 over it
    int live;           // its live tokens
};

// What a thread brings of a tile: N pieces of 16 bytes of each plane, of 4 * D. Key
// piece u: token u / (D / 16), channels 16 * (u % (D / 16)) ..; value piece u:
// strip u / D, channel u % D. Both planes' pieces u lie in strip u / D of the tile,
// which is one strip for a wave: pages and addresses are scalars.
template <int D, int INT8, int W>
struct Stage {
    static constexpr int kThreads = 64 * W, kPieces = 4 * D;
    static constexpr int N = kPieces / kThreads;
    static_assert(kPieces % kThreads == 0, "every thread brings N pieces");
    u4_t k[N], v[N];
    int live[N];   // live tokens of the pieces' strips
    int32_t e[N];  // the next fetch's block-table entries, as they come from memory
    int32_t es;    // lanes 0 to 3 of the first wave: the same of strip `lane`, its
    float ks, vs;  // scales and live tokens
    int own;
    uint32_t zero;  // 0, in a vector register

    __device__ __forceinline__ Stage() { asm("v_mov_b32 %0, 0" : "=v"(zero)); }

    static __device__ __forceinline__ uint32_t piece(int r) { return r * kThreads + threadIdx.x; }
    static __device__ __forceinline__ uint32_t strip_of(int r)
    {
        return __builtin_amdgcn_readfirstlane(piece(r) / D);
    }
    static __device__ __forceinline__ bool first_wave()
    {
        return __builtin_amdgcn_readfirstlane(threadIdx.x / 64) == 0;
    }
    // (past the table lies past the context too)
    static __device__ __forceinline__ int live_of(const Kv8AttnParams& p, int32_t e, uint32_t L,
                                                  uint32_t strip)
    {
        const int left = (int)L - (int)(16 * strip);
        return e < 0 || (uint32_t)e >= p.P || left < 0 ? 0 : left > 16 ? 16 : left;
    }
    static __device__ __forceinline__ uint32_t page_of(const Kv8AttnParams& p, int32_t e)
    {
        return e < 0 || (uint32_t)e >= p.P ? 0u : (uint32_t)e;
    }

    static __device__ __forceinline__ uint32_t index(const Kv8AttnParams& p, Divisor per_page,
                                                     uint32_t strip)
    {
        const uint32_t i = div_by(strip, per_page);
        return i < p.M ? i : p.M - 1;
    }
    // Nothing here looks at what it loads: that would wait for it, once a tile.
    __device__ __forceinline__ void entries(const Kv8AttnParams& p, const int32_t* table,
                                            Divisor per_page, uint32_t t0)
    {
        // (a vector load, though one entry a wave: a scalar one is waited for together
        // with the wave's LDS reads)
#pragma unroll
        for (int r = 0; r < N; ++r)
            e[r] = table[index(p, per_page, t0 / 16 + strip_of(r)) + zero];
        if (first_wave()) es = table[index(p, per_page, t0 / 16 + (threadIdx.x & 3u))];
    }
    __device__ __forceinline__ void fetch(const Kv8AttnParams& p, Divisor per_page, uint32_t h,
                                          uint32_t L, uint32_t t0)
    {
#pragma unroll
        for (int r = 0; r < N; ++r) {
            const uint32_t u = piece(r), strip = t0 / 16 + strip_of(r);
            const int32_t entry = __builtin_amdgcn_readfirstlane(e[r]);
            const uint32_t in = strip - div_by(strip, per_page) * (p.S / 16);
            const uint64_t at = (((uint64_t)page_of(p, entry) * p.Hkv + h) * p.S + in * 16) * D;
            // a strip's keys and values are 16 * D consecutive bytes, its pieces in order
            k[r] = *(const u4_t*)(p.key_cache + at + 16 * (u % D));
            v[r] = *(const u4_t*)(p.value_cache + at + 16 * (u % D));
            live[r] = live_of(p, entry, L, strip);
        }
        if (first_wave()) {
            const uint64_t row = (uint64_t)page_of(p, es) * p.Hkv + h;
            ks = p.scales[row];
            vs = p.scales[(uint64_t)p.P * p.Hkv + row];
            own = live_of(p, es, L, t0 / 16 + (threadIdx.x & 3u));
        }
    }
    // AGAIN: take_nan from the tile's values, whose first token is `token`.
    template <int AGAIN>
    __device__ __forceinline__ void store(char* tile, StripInfo* info, uint32_t* first_nan,
                                          uint32_t token) const
    {
#pragma unroll
        for (int r = 0; r < N; ++r) {
            const uint32_t u = piece(r);
            {
                const uint32_t token = u / (D / 16), block = token / 32, x = token % 32;
                const uint32_t m = (x & 16) | (x & 4) << 1 | (x & 8) >> 1 | (x & 3);
                char* to = tile + (block * (D / 16) + u % (D / 16)) * Tile<D>::kKeyBlock + m * 16;
                *(h8_t*)to = widen8<INT8>(k[r][0], k[r][1]);
                *(h8_t*)(to + 512) = widen8<INT8>(k[r][2], k[r][3]);
            }
            {
                // a dead token's bytes may be a NaN: 0 times it is not 0
                u4_t w = v[r];
                if (live[r] < 16) w = live_bytes(w, live[r]);
                const uint32_t strip = u / D, c = u % D;
                if constexpr (AGAIN) take_nan(w, token + 16 * strip, &first_nan[c]);
                char* to = tile + Tile<D>::kKeys + (strip * (D / 32) + c / 32) * 1024 + (c % 32) * 16;
                *(h8_t*)to = widen8<INT8>(w[0], w[1]);
                *(h8_t*)(to + 512) = widen8<INT8>(w[2], w[3]);
            }
        }
        if (threadIdx.x < kStrips) {
            StripInfo i;
            i.ks = held_scale(ks);
            const float s = held_scale(vs);
            i.lv = __builtin_amdgcn_logf(s);
            i.rvs = 0x1.0p+8f * __builtin_amdgcn_rcpf(s);
            i.live = own;
            info[threadIdx.x] = i;
        }
    }
};

// The token tiles that some row of a row tile sees, and those of each of its K
// parts.
struct Span {
    uint32_t tiles, each;

    __device__ __forceinline__ Span(const Kv8AttnParams& p, const SequenceBase& seq, uint32_t f0,
                                    uint32_t rows)
    {
        uint32_t end = seq.tokens;
        if (p.causal) {
            const uint32_t all = seq.rows * p.G, last = f0 + rows < all ? f0 + rows - 1 : all - 1;
            const int64_t x = (int64_t)seq.tokens - seq.all + last / p.G + 1;
            end = x < 0 ? 0u : (uint32_t)x;
        }
        tiles = (end + kTile - 1) / kTile;
        each = (tiles + p.K - 1) / p.K;
    }
};

template <int D, int BF16, int INT8, int W>
__global__ __launch_bounds__(64 * W, D < 256 ? 2 : 1) void kv8_prefill(Kv8AttnParams p,
                                                                       Divisor per_page)
{
    constexpr int KK = D / 16, CB = D / 32;
    __shared__ __align__(16) char lds[2 * Tile<D>::kBytes];
    __shared__ StripInfo info[2][kStrips];
    __shared__ uint32_t first_nan[D];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, n = lane & 31u, half = lane >> 5;

    // the heads of a tile lie next to each other in the grid (one an XCD, where
    // there are eight), then the parts of its tokens; a sequence's last tiles, the
    // longest, come first
    const uint32_t h = blockIdx.x % p.Hkv, part = blockIdx.x / p.Hkv % p.K;
    uint32_t t = gridDim.x / (p.Hkv * p.K) - 1 - blockIdx.x / (p.Hkv * p.K), b = 0;
    SequenceBase seq;
    {
        uint32_t before = 0;
        for (uint32_t b0 = 0;; b0 += 64) {
            if (b0 >= p.B) return;
            uint32_t tiles = 0;
            SequenceBase mine;
            if (b0 + lane < p.B) {
                mine = SequenceBase(p, b0 + lane);
                tiles = (mine.rows * p.G + group_rows(W) - 1) / group_rows(W);
            }
            const uint32_t upto = before + wave_scan(tiles);
            const uint64_t past = __ballot(upto > t);
            if (past) {
                const uint32_t l = (uint32_t)__builtin_ctzll(past);
                b = b0 + l;
                seq = mine.of_lane(l);
                t -= __builtin_amdgcn_readlane(upto - tiles, l);
                break;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    const uint32_t f0 = t * group_rows(W), all_rows = seq.rows * p.G;
    const int32_t* table = p.tables + (uint64_t)b * p.M;

    // the lane's row, and the tokens before `limit` that it sees
    const uint32_t f = f0 + wave * 32 + n, fr = f < all_rows ? f : all_rows - 1;
    int32_t limit = (int32_t)seq.tokens;
    if (p.causal) {
        const int64_t x = (int64_t)seq.tokens - seq.all + fr / p.G + 1;
        limit = x < 0 ? 0 : (int32_t)x;
    }
    h8_t q[KK];
    float qf, l;
    References ref;
    f16_t o[CB];
    {
        uint32_t row = seq.row0 + fr / p.G;
        if (row >= p.rows) row = p.rows - 1;
        const uint16_t* src = (const uint16_t*)p.q + (uint64_t)row * p.q_stride +
                              (uint64_t)(h * p.G + fr % p.G) * D + 8 * half;
        u4_t raw[KK];
#pragma unroll
        for (int k = 0; k < KK; ++k) raw[k] = *(const u4_t*)(src + 16 * k);
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < KK * 8; ++i) {
            const uint32_t w = raw[i / 8][(i / 2) & 3];
            most = fmaxf(most, fabsf(widen_el<BF16>((i & 1) ? w >> 16 : w & 0xffffu)));
        }
        most = fmaxf(most, xor_lanes(most, 32));
        const float shift = row_shift(most);
        qf = (1.0f / shift) * (fabsf(p.scale) * kLog2e);
        // a negative scale turns the row, so that larger products are larger scores; one
        // that is no number makes it such (fac is held at its least below)
        const float turned = p.scale < 0.0f ? -shift : p.scale == p.scale ? shift : p.scale;
#pragma unroll
        for (int i = 0; i < KK * 8; ++i) {
            const uint32_t w = raw[i / 8][(i / 2) & 3];
            q[i / 8][i % 8] = (_Float16)(widen_el<BF16>((i & 1) ? w >> 16 : w & 0xffffu) * turned);
        }
    }

    // tokens that every row of the wave sees, and that some row does
    int32_t whole = (int32_t)seq.tokens, some = (int32_t)seq.tokens;
    if (p.causal) {
        const uint32_t wf = f0 + wave * 32;
        const int64_t y = (int64_t)seq.tokens - seq.all + wf / p.G + 1;
        whole = y < 0 ? 0 : y < seq.tokens ? (int32_t)y : (int32_t)seq.tokens;
        const int64_t z = (int64_t)seq.tokens - seq.all + (wf + 31) / p.G + 1;
        some = z < 0 ? 0 : z < seq.tokens ? (int32_t)z : (int32_t)seq.tokens;
    }
    if (f0 + wave * 32 >= all_rows) some = 0;  // no row of its own
    const Span span(p, seq, f0, group_rows(W));
    const uint32_t first = part * span.each;
    if (part && first >= span.tiles) return;
    const uint32_t end = first + span.each < span.tiles ? first + span.each : span.tiles;

    // The walk. A causal one that ends with a NaN among its sums is made `again`, without
    // the NaN among the values' codes (take_nan); a test for them at the causal edge, in
    // one walk for all calls, costs up to 5% by the registers that it holds.
    auto walk = [&](auto again) __attribute__((always_inline)) {
        constexpr int AGAIN = decltype(again)::value;
        float gap = 0.0f;
        l = 0.0f;
        ref = References::none();
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
        Stage<D, INT8, W> stage;
        if (first < end) {
            stage.entries(p, table, per_page, first * kTile);
            stage.fetch(p, per_page, h, seq.tokens, first * kTile);
            stage.template store<AGAIN>(lds + (first & 1) * Tile<D>::kBytes, info[first & 1],
                                        first_nan, first * kTile);
        }
        if (first + 1 < end) {
            stage.entries(p, table, per_page, (first + 1) * kTile);
            stage.fetch(p, per_page, h, seq.tokens, (first + 1) * kTile);
            stage.entries(p, table, per_page, (first + 2) * kTile);
        }
        for (uint32_t j = first; j < end; ++j) {
            __syncthreads();  // tile j is in LDS, the other buffer has been read
            char* tile = lds + (j & 1) * Tile<D>::kBytes;
            const StripInfo* at = info[j & 1];
            const int32_t t0 = (int32_t)(j * kTile);
            if (j + 1 < end) {
                stage.template store<AGAIN>(lds + ((j + 1) & 1) * Tile<D>::kBytes,
                                            info[(j + 1) & 1], first_nan, t0 + kTile);
                if (j + 2 < end) {
                    // (the entries of tile j + 2 came a tile ago)
                    stage.fetch(p, per_page, h, seq.tokens, t0 + 2 * kTile);
                    stage.entries(p, table, per_page, t0 + 3 * kTile);
                }
            }
            if (t0 >= some) continue;

            // The tile's operand blocks in the order of their MFMA: the keys of both
            // blocks of tokens, then the values strip by strip. A ring of registers
            // holds the next kRing of them, or each MFMA would wait for its LDS read
            // (8192 rows of 32 heads of 128, when it was added: 616 us without, 597 with
            // four, 594 with eight; 256 channels leave registers for two: 865 us, 930
            // with four).
            constexpr int kRing = D == 256 ? 2 : 4, kScores = 2 * KK;
            h8_t ring[kRing];
            auto operand = [&](int i) {
                const int to = i < kScores ? i * Tile<D>::kKeyBlock
                                           : Tile<D>::kKeys + (i - kScores) * 1024;
                return *(const h8_t*)(tile + to + lane * 16);
            };
            f16_t s[2];
#pragma unroll
            for (int i = 0; i < kRing; ++i) ring[i] = operand(i);
            __builtin_amdgcn_sched_group_barrier(0x100, kRing, 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                s[i / KK] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], q[i % KK], s[i / KK],
                                                                   0, 0, 0);
                ring[i % kRing] = operand(i + kRing);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            StripInfo st[kStrips];
            int least = 16;
#pragma unroll
            for (int x = 0; x < kStrips; ++x) {
                st[x] = at[x];
                least = st[x].live < least ? st[x].live : least;
            }
            if (least < 16 || t0 + kTile > whole) {
                // token 8 half + i of strip x
#pragma unroll
                for (int x = 0; x < kStrips; ++x) {
                    const int ahead = limit - t0 - 16 * x;
                    const int sees = (ahead < st[x].live ? ahead : st[x].live) - (int)(8 * half);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float y = s[x / 2][8 * (x & 1) + i];
                        s[x / 2][8 * (x & 1) + i] = i < sees ? y : -__builtin_inff();
                    }
                }
            }
            float fac[kStrips], product = -__builtin_inff(), lv = st[0].lv;
            auto largest = [&](int x) {
                float y = s[x / 2][8 * (x & 1)];
#pragma unroll
                for (int i = 1; i < 8; ++i) y = fmaxf(y, s[x / 2][8 * (x & 1) + i]);
                return y;
            };
#pragma unroll
            for (int x = 0; x < kStrips; ++x) {
                // (not 0: a masked score is -inf)
                fac[x] = fmaxf(st[x].ks * qf, 1e-37f);
                product = fmaxf(product, __builtin_fmaf(largest(x), fac[x], st[x].lv));
                lv = fminf(lv, st[x].lv);
            }
            if (__any(ref.passes_or_holds(product, lv))) {
                float weight = largest(0) * fac[0];
#pragma unroll
                for (int x = 1; x < kStrips; ++x) weight = fmaxf(weight, largest(x) * fac[x]);
                product = fmaxf(product, xor_lanes(product, 32));
                weight = fmaxf(weight, xor_lanes(weight, 32));
                const References r = ref.moved_to(product, weight);
                l *= r.s;
#pragma unroll
                for (int c = 0; c < CB; ++c) o[c] *= r.m;
                gap = ref.gap();
#pragma unroll
                for (int x = 0; x < kStrips; ++x) ref.hold(st[x].lv, st[x].rvs);
            }
            h8_t pr[kStrips];
            float weights = 0.0f;
#pragma unroll
            for (int x = 0; x < kStrips; ++x) {
                const float off = st[x].lv - ref.m;
                float sum;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(s[x / 2][8 * (x & 1) + i], fac[x], off));
                    sum = i ? sum + e : e;
                    pr[x][i] = (_Float16)e;
                }
                weights += sum * st[x].rvs;
            }
            l += weights * gap;
#pragma unroll
            for (int i = 0; i < kScores; ++i) {
                const int c = i % CB;
                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % kRing], pr[i / CB], o[c], 0, 0, 0);
                if (i + kRing < kScores) ring[i % kRing] = operand(kScores + i + kRing);
            }
        }
    };
    walk(Const<0>());
    const bool nan_matters = !INT8 && p.causal;
    if (nan_matters) {
        bool some = false;
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) some |= o[c][i] != o[c][i];
        for (uint32_t i = threadIdx.x; i < D; i += 64 * W) first_nan[i] = kNoToken;
        if (__syncthreads_or(some)) {
            walk(Const<1>());
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const u4_t t = *(const u4_t*)&first_nan[32 * c + 8 * x + 4 * half];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (t[i] < (uint32_t)limit) o[c][4 * x + i] = __builtin_nanf("");
                }
        }
    }

    const uint32_t row = seq.row0 + f / p.G;
    l += xor_lanes(l, 32);
    if (f >= all_rows || row >= p.rows) return;
    const uint64_t to = (uint64_t)row * p.Hq + h * p.G + f % p.G;
    if (span.each < span.tiles) {
        const uint64_t rec = to * p.K + part;
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *(f4_t*)(p.acc + rec * D + 32 * c + 8 * x + 4 * half) =
                    f4_t{o[c][4 * x], o[c][4 * x + 1], o[c][4 * x + 2], o[c][4 * x + 3]};
        if (half == 0) *(f4_t*)(p.stats + kKv8Stats * rec) = f4_t{ref.m, ref.s, l, 0.0f};
        return;
    }
    const Quotient y(ref, l);
    uint16_t* out = (uint16_t*)p.out + to * D + 4 * half;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *(u2_t*)(out + 32 * c + 8 * x) =
                u2_t{narrow2<BF16>(y(o[c][4 * x]), y(o[c][4 * x + 1])),
                     narrow2<BF16>(y(o[c][4 * x + 2]), y(o[c][4 * x + 3]))};
}

// The parts of the rows, joined: D / 4 lanes a (row, head), as many workgroups as a
// launch carries without their number counting (32000 rows x heads on a wave each
// took 32 us, 4 ns a workgroup).
constexpr uint32_t kJoinGroups = 1024;

template <int D, int BF16, int W>
__global__ __launch_bounds__(256) void kv8_prefill_combine(Kv8AttnParams p)
{
    constexpr uint32_t kLanes = D / 4, kPer = 256 / kLanes;
    const uint64_t all = (uint64_t)p.rows * p.Hq;
    const uint32_t ch = threadIdx.x % kLanes * 4;
    for (uint64_t at = (uint64_t)blockIdx.x * kPer + threadIdx.x / kLanes; at < all;
         at += (uint64_t)gridDim.x * kPer) {  // row * Hq + head
        const uint32_t row = (uint32_t)(at / p.Hq), hq = (uint32_t)(at % p.Hq);
        const uint32_t b = sequence_of(p, row);
        if (b >= p.B) continue;
        const SequenceBase s(p, b);
        if (row < s.row0 || row - s.row0 >= s.rows) continue;
        const uint32_t f = (row - s.row0) * p.G + hq % p.G;
        const Span span(p, s, f / group_rows(W) * group_rows(W), group_rows(W));
        if (span.each >= span.tiles) continue;  // one part: it went to the output
        const uint32_t parts = (span.tiles + span.each - 1) / span.each;
        const float* stats = p.stats + kKv8Stats * at * p.K;
        // eight parts' loads at a time (past the last: its own again, left out)
        References ref = References::none();
        float l = 0.0f;
        f4_t a = {0, 0, 0, 0};
        for (uint32_t k0 = 0; k0 < parts; k0 += 8) {
            f4_t st[8];
            f4_t x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = k0 + j < parts ? k0 + j : parts - 1;
                st[j] = *(const f4_t*)(stats + kKv8Stats * k);
                x[j] = *(const f4_t*)(p.acc + (at * p.K + k) * D + ch);
            }
            const References was = ref;
#pragma unroll
            for (int j = 0; j < 8; ++j) ref = {fmaxf(ref.m, st[j][0]), fmaxf(ref.s, st[j][1])};
            l *= __builtin_amdgcn_exp2f(was.s - ref.s);
            a *= __builtin_amdgcn_exp2f(was.m - ref.m);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (k0 + j >= parts) break;
                l += __builtin_amdgcn_exp2f(st[j][1] - ref.s) * st[j][2];
                a += __builtin_amdgcn_exp2f(st[j][0] - ref.m) * x[j];
            }
        }
        const Quotient y(ref, l);
        *(u2_t*)((uint16_t*)p.out + at * D + ch) =
            u2_t{narrow2<BF16>(y(a[0]), y(a[1])), narrow2<BF16>(y(a[2]), y(a[3]))};
    }
}

template <int D, int BF16, int INT8, int W>
hipError_t launch_t(hipStream_t stream, const Kv8AttnParams& p)
{
    // at most so many tiles: whole ones of all rows, and one more a sequence
    const uint64_t rows = (uint64_t)p.rows * p.G;
    const uint64_t tiles = rows / group_rows(W) + (p.B < rows ? p.B : rows);
    hipLaunchKernelGGL((kv8_prefill<D, BF16, INT8, W>), dim3((uint32_t)(tiles * p.K * p.Hkv)),
                       dim3(64 * W), 0, stream, p, div_magic(p.S / 16));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.K == 1) return e;
    const uint64_t joins = ((uint64_t)p.rows * p.Hq * (D / 4) + 255) / 256;
    hipLaunchKernelGGL((kv8_prefill_combine<D, BF16, W>),
                       dim3(joins < kJoinGroups ? (uint32_t)joins : kJoinGroups), dim3(256), 0,
                       stream, p);
    return hipGetLastError();
}

template <int D, int BF16, int INT8>
hipError_t launch_w(hipStream_t stream, const Kv8AttnParams& p)
{
    if constexpr (D == 128) {
        if (kv8_prefill_waves(D, (uint64_t)p.max_q * p.G, (uint64_t)p.M * p.S) == 8)
            return launch_t<D, BF16, INT8, 8>(stream, p);
    }
    return launch_t<D, BF16, INT8, 4>(stream, p);
}

template <int D>
hipError_t launch_d(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p)
{
    if (bf16) return int8 ? launch_w<D, 1, 1>(stream, p) : launch_w<D, 1, 0>(stream, p);
    return int8 ? launch_w<D, 0, 1>(stream, p) : launch_w<D, 0, 0>(stream, p);
}

}  // namespace

hipError_t launch_kv8_prefill(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p)
{
    switch (p.D) {
        case 64: return launch_d<64>(stream, bf16, int8, p);
        case 128: return launch_d<128>(stream, bf16, int8, p);
        case 256: return launch_d<256>(stream, bf16, int8, p);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace tq4
