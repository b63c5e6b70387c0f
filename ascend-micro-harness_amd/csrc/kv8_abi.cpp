// kv8_abi.cpp -- the C ABI of the 8-bit paged cache (include/tq4_kv8.h): host
// checks, split counts and launches.
#include <hip/hip_runtime.h>

#include "../../include/tq4.h"
#include "../../include/tq4_kv8.h"
#include "kv8_internal.hpp"

namespace {

constexpr uint32_t kStrip = 16;
constexpr uint32_t kMaxPage = 1024;  // the writer's LDS map of a page's rows

// A launch holds fewer than 2^32 work-items: so many workgroups of 256.
constexpr uint64_t kMaxGroups = 0xffffffu;

int launched(hipError_t e) { return e == hipSuccess ? TQ4_OK : TQ4_ERR_LAUNCH; }

bool aligned(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// a * b * c held at 2^64 - 1
uint64_t mul(uint64_t a, uint64_t b, uint64_t c = 1)
{
    uint64_t r;
    if (__builtin_mul_overflow(a, b, &r) || __builtin_mul_overflow(r, c, &r)) return ~0ull;
    return r;
}

int cache_checks(int element_type, int code_type, uint32_t num_kv_heads, uint32_t head_size,
                 uint32_t block_size, uint32_t num_blocks)
{
    if (head_size != 64 && head_size != 128 && head_size != 256) return TQ4_ERR_HEAD_SIZE;
    if ((element_type != 0 && element_type != 1) ||
        (code_type != TQ4_KV8_FP8 && code_type != TQ4_KV8_INT8) || num_kv_heads == 0 ||
        num_blocks == 0 || block_size == 0 || block_size % kStrip || block_size > kMaxPage)
        return TQ4_ERR_GEOMETRY;
    // slots are 32-bit; pages and heads are indexed in 32 bits too
    if (mul(num_blocks, block_size) > 0x80000000ull || mul(num_blocks, num_kv_heads, 2) > 0xffffffffull)
        return TQ4_ERR_RANGE;
    return TQ4_OK;
}

// How a call's work is cut (kv8_decode.hip): K parts a sequence, or 0: streamed
// over `groups` workgroups.
struct Cut {
    uint32_t K, groups;
};

uint64_t tiles_of(uint64_t max_q, uint64_t group)
{
    return (max_q * group + tq4::kKv8Rows - 1) / tq4::kKv8Rows;
}

// The choice between one workgroup an item (no second kernel), even parts, and
// streaming, which keeps all CUs busy whatever the lengths are. A workgroup walks cap
// tokens in cap * d * 0.0375 ns, all items together cost their bytes at 4.9 TB/s
// (3.9 with half the CUs) and a second kernel 4 us. Heads of 128, 8 KV heads, 4 rows
// each, tables as wide as the longest context, us for one workgroup / parts / streamed:
//   4 sequences of 300..1500 tokens   11.8 /  8.9 / 12.4
//   16 of 300..1500                   12.2 / 13.2 / 18.5
//   16 of 300..4099                   24.0 / 21.9 / 24.7
//   16 of 500..20000                  132  / 85   / 79     parts of 10000: uneven
//   32 of 500..4096                   35.4 / 40.8 / 36.9
//   128 of 500..4096                  131  / 133  / 121    (3000..4096: 172 / 182 / 176)
// cap is the table's tokens, so in a table far wider than its contexts the choice is
// that of longer ones (in one of 8192 tokens and more, 16 of 600..2048: 14.5 -> 19.7).
// Parts: one workgroup a CU (one sequence of 4096: 16 / 32 / 64 parts 9.4 / 9.0 / 9.9
// us; of 65536 32 / 64 31.5 / 32.4), of 128 of the table's tokens at least, and no more
// than 64, or 128, where the join's share grows (2 heads of 65536: 64 / 128 parts 15.2 /
// 15.5; of 256 channels 23.1 / 21.8).
Cut cut_rule(uint32_t d, uint64_t seqs, uint64_t heads, uint64_t tiles, uint64_t cap,
             uint32_t num_splits)
{
    Cut c{num_splits, 0};
    if (num_splits) return c;
    c.groups = 256u * (uint32_t)tq4::kKv8GroupsPerCu((int)d);
    uint64_t items = mul(seqs, heads, tiles);
    if (items == 0) items = 1;
    const uint64_t walk = mul(cap, d * 3ull) / 80, all = mul(mul(items, cap), d * 2ull) / 4900;
    uint64_t k = 256 / items;
    if (k > (cap + 127) / 128) k = (cap + 127) / 128;
    if (k > (d == 256 ? 128 : 64)) k = d == 256 ? 128 : 64;
    if (k > 1) {
        const uint64_t one = walk > all / 4 * 5 ? walk : all / 4 * 5;
        const uint64_t parts = (walk / k > all ? walk / k : all) + 4000;
        c.K = one <= parts ? 1 : seqs == 1 || walk / k <= 15000 ? (uint32_t)k : 0;
    } else if (seqs == 1 || (walk <= 20000 && walk <= all + 4500)) {
        c.K = 1;
    }
    return c;
}

uint32_t record_rows(uint64_t max_q, uint64_t group)
{
    return (uint32_t)(max_q * group < tq4::kKv8Rows ? max_q * group : tq4::kKv8Rows);
}

// Records of a call: (floats of a row's sums, and its statistics) a row and slot.
uint64_t record_slots(const Cut& c, uint64_t items)
{
    return c.K == 1 ? 0 : c.K ? mul(items, c.K) : 2ull * c.groups;
}
size_t record_bytes(const Cut& c, uint64_t items, uint32_t rec_rows, uint32_t d)
{
    const uint64_t b =
        mul(mul(record_slots(c, items), rec_rows), (uint64_t)d + tq4::kKv8Stats, sizeof(float));
    return b > (uint64_t)SIZE_MAX - 16 ? SIZE_MAX : (size_t)((b + 15) & ~15ull);
}

// Whether the decode kernel takes a prefill call: its tiles of 16 rows each read
// the context from L2, and are as many workgroups more, against tiles of 128 rows
// and more in LDS. Up to 32 rows it is the better; behind, while its tiles are at
// most three times those that the GPU holds at once, and its tiles times a table's
// tokens are few. Measured with 4 rows of 8 KV heads of 128 a token (us, decode
// kernel against the other; rows of a sequence and KV head):
//   32 rows   16 sequences of 500..4000 tokens  26, 40;   of 500..1000   11, 23
//   64 rows   the same                          44, 50;   17, 28
//   256 rows  the same                         156, 92;   47, 34
//   512 rows  4 sequences of 1000 tokens        27, 32;   1024 rows      45, 33
//   256 rows  1 sequence of 4096                19, 34;   of 32768       82, 63
// The product is no sharp line: at 2.0 million 1536 rows of one sequence of 2600 take
// 41, 46, but 192 rows of 4 of 5200 take 84, 41. Heads of 256: 256 rows of one of 4096
// (0.5 million) 33, 51; 64 rows of 16 of 500..1000 35, 57; 192 rows of one of 16384 (1.6
// million) 85, 76; 384 rows of 4 of 2600 (2.0 million) 154, 87.
bool few_rows(uint32_t d, uint64_t num_rows, uint64_t seqs, uint64_t heads, uint64_t group,
              uint64_t max_q, uint64_t cap)
{
    const uint64_t tiles = tiles_of(max_q, group);
    if (tiles <= 2) return true;
    uint64_t all = mul(seqs, tiles);
    if (all > num_rows * group / tq4::kKv8Rows + seqs) all = num_rows * group / tq4::kKv8Rows + seqs;
    all = mul(all, heads);
    return mul(heads, tiles) <= 65535u && all <= 768ull * tq4::kKv8GroupsPerCu((int)d) &&
           mul(all, cap) <= (d == 256 ? 1310720u : 2250000u);
}

// The parts that a prefill's row tiles cut their tokens into: with fewer row tiles
// than the CUs hold at once, as many as fill them, of 256 of the table's tokens at
// least and while a part's records (written and read: 8 bytes an element at 2.4 TB/s)
// cost less than it saves (a tile of 64 tokens is taken for 2.2 us with eight waves, 1.3
// with four). 1024 rows of 8 KV heads of 128 over 4096 tokens: 121 us in one part, 45 in
// 6, 43 in 8 (taken), 56 in 11; 512 over 16384: 450, 64 in 11 (taken), 58 in 16. Shorter
// contexts in a wide table have shorter parts (512 rows over 512 tokens: 8 us by the
// decode kernel in a table of 8192, 27 in one of 32768).
uint32_t prefill_parts(uint32_t d, uint64_t num_rows, uint64_t seqs, uint64_t heads,
                       uint64_t group, uint64_t max_q, uint64_t cap)
{
    const uint64_t waves = tq4::kv8_prefill_waves(d, max_q * group, cap), rows = 32 * waves;
    uint64_t tiles = mul(seqs, (max_q * group + rows - 1) / rows);
    if (tiles > mul(num_rows, group) / rows + seqs) tiles = mul(num_rows, group) / rows + seqs;
    const uint64_t groups = mul(tiles, heads);
    uint64_t k = groups ? tq4::kv8_prefill_fit(d, (uint32_t)waves) / groups : 1;
    if (k > cap / 256) k = cap / 256;
    const uint64_t saved = (waves == 8 ? 2200 : 1300) * (cap / tq4::kKv8Unit);  // ns
    const uint64_t cost = mul(mul(num_rows, group), heads, d * 8ull) / 2400 + 1;
    while (k > 1 && mul(k, k, cost) > saved) --k;
    return (uint32_t)(k < 1 ? 1 : k > 64 ? 64 : k);
}

// The grids and the line of a streamed call's units in bounds; `rows` output rows,
// each a workgroup of the join, of 1024 where there are many records.
bool cut_fits(const Cut& c, uint64_t seqs, uint64_t cap, uint64_t heads, uint64_t tiles,
              uint64_t rows)
{
    const uint32_t join = tq4::kv8_join_waves(c.K, c.groups, mul(seqs, heads, tiles));
    if (rows > (join == 16 ? kMaxGroups / 4 : kMaxGroups)) return false;
    if (c.K) return mul(seqs, c.K) <= kMaxGroups && mul(heads, tiles) <= 65535u;
    return mul(mul(seqs, (cap + tq4::kKv8Unit - 1) / tq4::kKv8Unit), heads, tiles) <= 0xff000000ull;
}

int attention_checks(const void* q, const void* kc, const void* vc, const float* sc,
                     const int32_t* tables, const int32_t* lens, const void* out,
                     uint64_t q_stride, uint32_t rows, uint32_t num_seqs, uint32_t num_heads,
                     uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                     uint32_t max_blocks)
{
    if (num_heads == 0 || num_heads % num_kv_heads || num_heads / num_kv_heads > 16 ||
        max_blocks == 0)
        return TQ4_ERR_GEOMETRY;
    if (mul(max_blocks, block_size) > 0x7fffffffull || rows > 0x7fffffffu ||
        num_seqs > 0x7fffffffu || num_kv_heads > 65535u)
        return TQ4_ERR_RANGE;
    if (!q || !kc || !vc || !sc || !tables || !lens || !out) return TQ4_ERR_NULL_POINTER;
    if (!aligned(q) || !aligned(kc) || !aligned(vc) || !aligned(out) || q_stride % 8)
        return TQ4_ERR_ALIGNMENT;
    if (rows > 1 && q_stride < (uint64_t)num_heads * head_size) return TQ4_ERR_GEOMETRY;
    return TQ4_OK;
}

tq4::Kv8AttnParams make(const void* q, const void* kc, const void* vc, const float* sc,
                        const int32_t* tables, const int32_t* lens, const int32_t* cu, void* out,
                        uint64_t q_stride, uint32_t rows, uint32_t num_seqs, uint32_t num_heads,
                        uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                        uint32_t num_blocks, uint32_t max_blocks, uint32_t max_q, int causal,
                        float scale, const Cut& cut, void* workspace)
{
    tq4::Kv8AttnParams p{};
    p.q = q;
    p.key_cache = (const uint8_t*)kc;
    p.value_cache = (const uint8_t*)vc;
    p.scales = sc;
    p.tables = tables;
    p.context_lens = lens;
    p.cu = cu;
    p.rec_rows = record_rows(max_q, num_heads / num_kv_heads);
    p.acc = (float*)workspace;
    const uint64_t items = (uint64_t)num_seqs * num_kv_heads *
                           tiles_of(max_q, num_heads / num_kv_heads);
    if (const uint64_t slots = record_slots(cut, items))
        p.stats = p.acc + slots * p.rec_rows * head_size;
    p.out = out;
    p.q_stride = q_stride;
    p.rows = rows;
    p.B = num_seqs;
    p.Hq = num_heads;
    p.Hkv = num_kv_heads;
    p.G = num_heads / num_kv_heads;
    p.D = head_size;
    p.S = block_size;
    p.P = num_blocks;
    p.M = max_blocks;
    p.K = cut.K;
    p.groups = cut.groups;
    p.max_q = max_q;
    p.causal = causal;
    p.scale = scale;
    return p;
}

}  // namespace

extern "C" {

size_t tq4_paged_plan_workspace_bytes(uint32_t num_requests)
{
    return tq4::plan_workspace_bytes(num_requests);
}

int tq4_paged_plan(void* stream, const int32_t* context_lens, const int32_t* query_lens,
                   const int32_t* release, int32_t* block_tables, int32_t* free_pages,
                   const int32_t* free_state, int32_t* slot_mapping, int32_t* positions,
                   int32_t* cu_seqlens, int32_t* granted, int32_t* new_context_lens,
                   int32_t* new_free_state, void* workspace, size_t workspace_bytes,
                   uint32_t num_requests, uint32_t max_blocks_per_seq, uint32_t block_size,
                   uint32_t num_blocks, uint32_t max_tokens)
{
    if (num_requests == 0 || max_blocks_per_seq == 0 || num_blocks == 0 || block_size == 0 ||
        block_size % kStrip)
        return TQ4_ERR_GEOMETRY;
    if (mul(num_blocks, block_size) > 0x80000000ull ||
        mul(num_requests, max_blocks_per_seq) > 0x7fffffffull || max_tokens > 0x7fffffffu)
        return TQ4_ERR_RANGE;
    if (!context_lens || !query_lens || !block_tables || !free_pages || !free_state ||
        (!slot_mapping && max_tokens) || !cu_seqlens || !granted || !new_context_lens || !new_free_state)
        return TQ4_ERR_NULL_POINTER;
    if (!workspace || !aligned(workspace) ||
        workspace_bytes < tq4_paged_plan_workspace_bytes(num_requests))
        return TQ4_ERR_WORKSPACE;
    tq4::PlanParams p{};
    p.context_lens = context_lens;
    p.query_lens = query_lens;
    p.release = release;
    p.tables = block_tables;
    p.ring = free_pages;
    p.state = free_state;
    p.slots = slot_mapping;
    p.positions = positions;
    p.cu = cu_seqlens;
    p.granted = granted;
    p.new_lens = new_context_lens;
    p.new_state = new_free_state;
    p.ws = (int32_t*)workspace;
    p.B = num_requests;
    p.M = max_blocks_per_seq;
    p.S = block_size;
    p.P = num_blocks;
    p.T = max_tokens;
    return launched(tq4::launch_plan((hipStream_t)stream, p));
}

int tq4_kv8_reshape_and_cache(void* stream, int element_type, int code_type, const void* key,
                              const void* value, void* key_cache, void* value_cache,
                              float* scale_cache, const int32_t* slot_mapping,
                              uint64_t key_stride, uint64_t value_stride, uint32_t num_tokens,
                              uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                              uint32_t num_blocks)
{
    const int rc = cache_checks(element_type, code_type, num_kv_heads, head_size, block_size,
                                num_blocks);
    if (rc != TQ4_OK) return rc;
    if (num_tokens == 0) return TQ4_OK;
    if (num_kv_heads > 8192u || mul(num_tokens, num_kv_heads) > (1u << 26)) return TQ4_ERR_RANGE;
    if (!key || !value || !key_cache || !value_cache || !scale_cache || !slot_mapping)
        return TQ4_ERR_NULL_POINTER;
    if (!aligned(key) || !aligned(value) || !aligned(key_cache) || !aligned(value_cache) ||
        key_stride % 8 || value_stride % 8)
        return TQ4_ERR_ALIGNMENT;
    const uint64_t row = (uint64_t)num_kv_heads * head_size;
    if (num_tokens > 1 && (key_stride < row || value_stride < row)) return TQ4_ERR_GEOMETRY;
    tq4::Kv8WriteParams p{};
    p.key = key;
    p.value = value;
    p.key_cache = (uint8_t*)key_cache;
    p.value_cache = (uint8_t*)value_cache;
    p.scales = scale_cache;
    p.slots = slot_mapping;
    p.key_stride = key_stride;
    p.value_stride = value_stride;
    p.T = num_tokens;
    p.H = num_kv_heads;
    p.D = head_size;
    p.S = block_size;
    p.P = num_blocks;
    return launched(tq4::launch_kv8_writer((hipStream_t)stream, element_type,
                                           code_type == TQ4_KV8_INT8, p));
}

size_t tq4_kv8_decode_workspace_bytes(uint32_t num_seqs, uint32_t num_heads,
                                      uint32_t num_kv_heads, uint32_t head_size,
                                      uint32_t block_size, uint32_t max_blocks_per_seq,
                                      uint32_t num_splits)
{
    if (num_kv_heads == 0) return 0;
    const Cut c = cut_rule(head_size, num_seqs, num_kv_heads, 1,
                           (uint64_t)max_blocks_per_seq * block_size, num_splits);
    return record_bytes(c, (uint64_t)num_seqs * num_kv_heads,
                        record_rows(1, num_heads / num_kv_heads), head_size);
}

int tq4_kv8_paged_decode(void* stream, int element_type, int code_type, const void* q,
                         const void* key_cache, const void* value_cache,
                         const float* scale_cache, const int32_t* block_tables,
                         const int32_t* context_lens, void* workspace, size_t workspace_bytes,
                         void* out, uint64_t q_stride, uint32_t num_seqs, uint32_t num_heads,
                         uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                         uint32_t num_blocks, uint32_t max_blocks_per_seq, uint32_t num_splits,
                         float scale)
{
    int rc = cache_checks(element_type, code_type, num_kv_heads, head_size, block_size, num_blocks);
    if (rc != TQ4_OK) return rc;
    if (num_seqs == 0) return TQ4_OK;
    rc = attention_checks(q, key_cache, value_cache, scale_cache, block_tables, context_lens, out,
                          q_stride, num_seqs, num_seqs, num_heads, num_kv_heads, head_size,
                          block_size, max_blocks_per_seq);
    if (rc != TQ4_OK) return rc;
    if (num_splits > TQ4_KV8_MAX_SPLITS) return TQ4_ERR_SPLITS;
    const uint64_t cap = (uint64_t)max_blocks_per_seq * block_size;
    const Cut s = cut_rule(head_size, num_seqs, num_kv_heads, 1, cap, num_splits);
    if (!cut_fits(s, num_seqs, cap, num_kv_heads, 1, mul(num_seqs, num_heads)))
        return TQ4_ERR_RANGE;
    const size_t need = tq4_kv8_decode_workspace_bytes(num_seqs, num_heads, num_kv_heads, head_size,
                                                       block_size, max_blocks_per_seq, num_splits);
    if (need && (!workspace || !aligned(workspace) || workspace_bytes < need))
        return TQ4_ERR_WORKSPACE;
    return launched(tq4::launch_kv8_decode(
        (hipStream_t)stream, element_type, code_type == TQ4_KV8_INT8,
        make(q, key_cache, value_cache, scale_cache, block_tables, context_lens, nullptr, out,
             q_stride, num_seqs, num_seqs, num_heads, num_kv_heads, head_size, block_size,
             num_blocks, max_blocks_per_seq, 1, 0, scale, s, workspace)));
}

size_t tq4_kv8_prefill_workspace_bytes(uint32_t num_rows, uint32_t num_seqs, uint32_t num_heads,
                                       uint32_t num_kv_heads, uint32_t head_size,
                                       uint32_t block_size, uint32_t max_blocks_per_seq,
                                       uint32_t max_query_len)
{
    if (num_kv_heads == 0) return 0;
    if (max_query_len > num_rows) max_query_len = num_rows;
    const uint64_t group = num_heads / num_kv_heads, cap = (uint64_t)max_blocks_per_seq * block_size;
    if (!few_rows(head_size, num_rows, num_seqs, num_kv_heads, group, max_query_len, cap)) {
        const uint32_t k = prefill_parts(head_size, num_rows, num_seqs, num_kv_heads, group,
                                         max_query_len, cap);
        return k == 1 ? 0 : record_bytes(Cut{k, 0}, mul(num_rows, num_heads), 1, head_size);
    }
    const Cut c =
        cut_rule(head_size, num_seqs, num_kv_heads, tiles_of(max_query_len, group), cap, 0);
    return record_bytes(c, mul(num_seqs, num_kv_heads, tiles_of(max_query_len, group)),
                        record_rows(max_query_len, group), head_size);
}

int tq4_kv8_paged_prefill(void* stream, int element_type, int code_type, const void* q,
                          const void* key_cache, const void* value_cache,
                          const float* scale_cache, const int32_t* block_tables,
                          const int32_t* context_lens, const int32_t* cu_seqlens,
                          void* workspace, size_t workspace_bytes, void* out, uint64_t q_stride,
                          uint32_t num_rows, uint32_t num_seqs, uint32_t num_heads,
                          uint32_t num_kv_heads, uint32_t head_size, uint32_t block_size,
                          uint32_t num_blocks, uint32_t max_blocks_per_seq,
                          uint32_t max_query_len, int causal, float scale)
{
    int rc = cache_checks(element_type, code_type, num_kv_heads, head_size, block_size, num_blocks);
    if (rc != TQ4_OK) return rc;
    if (num_seqs == 0 || num_rows == 0 || max_query_len == 0) return TQ4_OK;
    rc = attention_checks(q, key_cache, value_cache, scale_cache, block_tables, context_lens, out,
                          q_stride, num_rows, num_seqs, num_heads, num_kv_heads, head_size,
                          block_size, max_blocks_per_seq);
    if (rc != TQ4_OK) return rc;
    if (!cu_seqlens) return TQ4_ERR_NULL_POINTER;
    if (max_query_len > num_rows) max_query_len = num_rows;
    const uint64_t group = num_heads / num_kv_heads, tiles = tiles_of(max_query_len, group);
    const uint64_t cap = (uint64_t)max_blocks_per_seq * block_size, rows = (uint64_t)num_rows * group;
    auto args = [&](const Cut& c) {
        return make(q, key_cache, value_cache, scale_cache, block_tables, context_lens, cu_seqlens,
                    out, q_stride, num_rows, num_seqs, num_heads, num_kv_heads, head_size,
                    block_size, num_blocks, max_blocks_per_seq, max_query_len, causal != 0, scale,
                    c, workspace);
    };
    const size_t need =
        tq4_kv8_prefill_workspace_bytes(num_rows, num_seqs, num_heads, num_kv_heads, head_size,
                                        block_size, max_blocks_per_seq, max_query_len);
    const bool room = !need || (workspace && aligned(workspace) && workspace_bytes >= need);
    if (!few_rows(head_size, num_rows, num_seqs, num_kv_heads, group, max_query_len, cap)) {
        const uint32_t k = prefill_parts(head_size, num_rows, num_seqs, num_kv_heads, group,
                                         max_query_len, cap);
        if (mul(mul(rows / 128 + num_seqs, num_kv_heads), k) > kMaxGroups / 2 ||
            mul(num_rows, num_heads) > kMaxGroups)
            return TQ4_ERR_RANGE;
        if (!room) return TQ4_ERR_WORKSPACE;
        tq4::Kv8AttnParams p = args(Cut{k, 0});
        p.stats = p.acc + (uint64_t)num_rows * num_heads * k * head_size;
        return launched(tq4::launch_kv8_prefill((hipStream_t)stream, element_type,
                                                code_type == TQ4_KV8_INT8, p));
    }
    const Cut s = cut_rule(head_size, num_seqs, num_kv_heads, tiles, cap, 0);
    if (!cut_fits(s, num_seqs, cap, num_kv_heads, tiles, mul(num_rows, num_heads)))
        return TQ4_ERR_RANGE;
    if (!room) return TQ4_ERR_WORKSPACE;
    return launched(tq4::launch_kv8_decode((hipStream_t)stream, element_type,
                                           code_type == TQ4_KV8_INT8, args(s)));
}

}  // extern "C"
