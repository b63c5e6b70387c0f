// kv8_internal.hpp -- launches of the 8-bit paged cache's kernels (tq4_kv8.h),
// called by kv8_abi.cpp after its checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tq4 {

constexpr float kKv8LeastScale = 0x1.0p-100f;
constexpr float kKv8MostScale = 0x1.0p+122f;  // 127 times it holds every BF16 value

struct PlanParams {
    const int32_t *context_lens, *query_lens, *release;
    int32_t *tables, *ring;
    const int32_t* state;
    int32_t *slots, *positions, *cu, *granted, *new_lens, *new_state;
    int32_t* ws;
    uint32_t B, M, S, P, T;
};
size_t plan_workspace_bytes(uint32_t B);
hipError_t launch_plan(hipStream_t stream, const PlanParams& p);

struct Kv8WriteParams {
    const void *key, *value;
    uint8_t *key_cache, *value_cache;
    float* scales;
    const int32_t* slots;
    uint64_t key_stride, value_stride;
    uint32_t T, H, D, S, P;
};
hipError_t launch_kv8_writer(hipStream_t stream, int bf16, int int8, const Kv8WriteParams& p);

// Attention; cu NULL: one row a sequence.
constexpr uint32_t kKv8Unit = 64, kKv8Rows = 16;  // tokens of a step, rows of a tile
constexpr uint32_t kKv8Stats = 4;  // of a record's row: its References, its sum, one unused
// Workgroups of the decode that a CU holds at once, by registers.
constexpr int kKv8GroupsPerCu(int d) { return d == 256 ? 1 : d == 128 ? 2 : 4; }

struct Kv8AttnParams {
    const void* q;
    const uint8_t *key_cache, *value_cache;
    const float* scales;
    const int32_t *tables, *context_lens, *cu;
    float *acc, *stats;  // records: [slot][rec_rows][D] and [slot][rec_rows][kKv8Stats]
    void* out;
    uint64_t q_stride;
    uint32_t rows, B, Hq, Hkv, G, D, S, P, M;
    uint32_t K;       // parts of a sequence; 0: streamed over `groups`
    uint32_t groups;  // workgroups
    uint32_t rec_rows;
    uint32_t max_q;
    int causal;
    float scale;
};
// Waves of a prefill workgroup, 32 rows each (kv8_prefill.hip), for so many rows of a
// (sequence, kv head) over tables of `cap` tokens, and the workgroups that the CUs
// hold at once. Eight waves widen a tile for twice the rows (8192 rows x 32 heads of
// 128: 568 us, 605 with four; 4000 rows 151, 175), four are the more balanced where there
// are few tiles (3000 rows: 99 us, 101 with eight; 2048: 62, 68; 1000: 33, 37); a tile of
// 64 channels has pieces for four, and 256 channels fill a wave's registers and a CU's
// LDS with four.
inline uint32_t kv8_prefill_waves(uint32_t d, uint64_t rows, uint64_t cap)
{
    return d == 128 && rows > 128 && cap > 2048 ? 8 : 4;
}
inline uint32_t kv8_prefill_fit(uint32_t d, uint32_t waves)
{
    return 256u * (waves == 8 || d == 256 ? 1 : d == 128 ? 2 : 3);
}

// Waves that join a row's records, by those that an item has, were all alike (K or
// `groups` as in Kv8AttnParams): more where there are many (and then few rows). 128
// records of 32 rows x 256: 13.6 us with one load at a time and four waves.
inline uint32_t kv8_join_waves(uint32_t K, uint32_t groups, uint64_t items)
{
    const uint64_t records = K ? K : groups / items;
    return records > 32 ? 16 : records > 8 ? 4 : 1;
}

hipError_t launch_kv8_decode(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p);
hipError_t launch_kv8_prefill(hipStream_t stream, int bf16, int int8, const Kv8AttnParams& p);

}  // namespace tq4
