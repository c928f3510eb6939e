// kvcache_plan.cpp -- the step plan of the cache operators (host only, no device call).
//
// A plan is one array of int32 words that the operators' kernels read from device memory:
//   table   the block tables, one sequence after the other
//   slots   for each new token, its cache slot (block * block_size + offset)
//   pages   for each table entry, {first row of the read-back output, tokens in the block}
//   row tiles, row starts   the attention's work for few rows (KvTile, KvStart)
//   tile items              ... and for many (KvItem)
//   joins   which partial rows make up which output rows (KvJoin)
// Lengths, block ids and the write set are checked while it is built, so no kernel can be
// sent outside a pool by a plan, and the work is balanced over the whole batch.
#include "kvcache_plan.h"
#include "kv_internal.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>
#include <vector>

namespace {

int refuse(int code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return kvm_internal_error(code, buf);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Sequences' sums stay in int32 (words of the plan), with room for a tile's overhang.
constexpr int64_t kMaxTokens = (1ll << 31) - 4096;

// Workgroups of the kernel for few rows: as many as run at the same time, by the CUs' registers and LDS.  Fewer leave memory
// waiting, more only add joins (us, head_dim 128, 1, 2 and 4 a CU: 96.7, 89.0, 89.5 for 32 sequences of 1000, 32 heads, 110, 109,
// 112 for 8 of 20000, 8 heads; head_dim 64, 2, 3 and 4: 27.0, 24.9, 28.6 for 64 of 600, 12 heads).
int64_t most_groups(int64_t head_dim) { return kCus * (head_dim <= 64 ? 3 : 2); }

}  // namespace

uint64_t kvm_step_seal(const KvmStep &s)
{
    // a mix of the words before the seal: a plan filled by hand or half overwritten is refused
    static_assert(offsetof(KvmStep, seal) % 8 == 0, "the sealed part is whole words");
    uint64_t h = 0x9e3779b97f4a7c15ull, w;
    for (size_t i = 0; i < offsetof(KvmStep, seal); i += 8) {
        memcpy(&w, (const char *)&s + i, 8);
        h = (h ^ w) * 0xff51afd7ed558ccdull;
        h ^= h >> 29;
    }
    return h;
}

extern "C" {

int64_t kvm_plan_words(int64_t num_seqs, int64_t num_tokens, int64_t num_pages, int64_t num_heads, int64_t num_kv_heads)
{
    // what a plan may have at most, so that the sum below stays in 64 bits
    if (num_seqs < 0 || num_tokens < 0 || num_pages < 0 || std::max({num_seqs, num_tokens, num_pages}) > INT32_MAX ||
        num_heads < 1 || num_heads > (1 << 20) || num_kv_heads < 1 || num_kv_heads > num_heads)
        return refuse(KVM_EINVAL, "kvm_plan_words: a step of that size is not supported");
    const int64_t group = std::max<int64_t>(1, num_heads / num_kv_heads);
    const int64_t tiles = num_seqs + num_tokens * group / 16;            // one at least for each sequence
    const int64_t big = num_seqs + num_tokens * group / kTileRows;
    return 64 + num_pages * 3 + num_tokens + tiles * kTileWords + most_groups(16) * (kStartWords + kJoinWords) +
           (2 * big + kTileTarget) * ceil_div(num_kv_heads, kHeadBlock) * kItemWords + big * num_kv_heads * kJoinWords;
}

int kvm_plan_step(const int64_t *first_token, const int64_t *new_tokens, int64_t num_seqs, const int64_t *table,
                  const int64_t *table_len, int64_t num_blocks, int64_t block_size, int64_t num_heads,
                  int64_t num_kv_heads, int64_t head_dim, int32_t dtype, int32_t format, int32_t *words, int64_t capacity,
                  KvmStep *step)
try {
    if (!step || !words) return refuse(KVM_EINVAL, "kvm_plan_step: null output");
    if (num_seqs < 0 || (num_seqs > 0 && (!first_token || !new_tokens)))
        return refuse(KVM_EINVAL, "kvm_plan_step: bad sequence lists");
    if (dtype != KVM_F16 && dtype != KVM_BF16 && dtype != KVM_F32)
        return refuse(KVM_EINVAL, "kvm_plan_step: unknown dtype %d", dtype);
    if (format != KVM_CACHE_PLAIN && format != KVM_CACHE_E4M3) return refuse(KVM_EINVAL, "unknown pool format %d", format);
    if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0 || num_heads > (1 << 20))
        return refuse(KVM_EINVAL, "num_heads (%lld) must be a positive multiple of num_kv_heads (%lld)",
                      (long long)num_heads, (long long)num_kv_heads);
    if (head_dim < 16 || head_dim > KVM_MAX_HEAD_DIM || head_dim % 16 != 0)
        return refuse(KVM_EINVAL, "head_dim is %lld: the cache operators want a multiple of 16 up to %d",
                      (long long)head_dim, KVM_MAX_HEAD_DIM);
    const bool cached = num_blocks > 0;
    if (num_blocks < 0 || num_blocks > INT32_MAX) return refuse(KVM_EINVAL, "bad number of blocks %lld", (long long)num_blocks);
    if (cached) {
        if (block_size < 1 || block_size > 65536) return refuse(KVM_EINVAL, "block_size %lld is not in [1, 65536]", (long long)block_size);
        if (num_blocks * block_size > INT32_MAX)
            return refuse(KVM_EINVAL, "pools of more than 2^31 token slots are not supported");
        if (num_seqs > 0 && (!table_len || !table)) return refuse(KVM_EINVAL, "kvm_plan_step: null block table");
    }
    const int64_t group = num_heads / num_kv_heads;

    // ---- lengths and tables
    int64_t tokens = 0, kv_tokens = 0, pages = 0;
    bool all_new = true;
    for (int64_t s = 0; s < num_seqs; ++s) {
        const int64_t a = first_token[s], n = new_tokens[s];
        if (a < 0 || n < 0 || a > kMaxTokens || n > kMaxTokens)
            return refuse(KVM_ERANGE, "sequence %lld: first_token %lld, new_tokens %lld", (long long)s, (long long)a, (long long)n);
        if (a > 0) all_new = false;
        tokens += n;
        kv_tokens += a + n;
        if (cached) {
            if (table_len[s] < 0) return refuse(KVM_ERANGE, "sequence %lld: negative table length", (long long)s);
            if (table_len[s] * block_size < a + n)
                return refuse(KVM_ERANGE, "sequence %lld has %lld tokens but its block table holds %lld blocks of %lld",
                              (long long)s, (long long)(a + n), (long long)table_len[s], (long long)block_size);
            pages += table_len[s];
        }
        if (tokens * group > kMaxTokens || kv_tokens > kMaxTokens || pages > kMaxTokens / 2)
            return refuse(KVM_EINVAL, "a step of more than 2^31 rows, cached tokens or blocks is not supported");
    }
    if (!cached && !all_new) return refuse(KVM_EINVAL, "a plan without a cache takes new sequences only");

    KvmStep out;
    memset(&out, 0, sizeof out);
    out.num_seqs = num_seqs;
    out.num_tokens = tokens;
    out.num_kv_tokens = kv_tokens;
    out.num_pages = pages;
    out.num_blocks = num_blocks;
    out.block_size = cached ? block_size : 0;
    out.num_heads = num_heads;
    out.num_kv_heads = num_kv_heads;
    out.head_dim = head_dim;
    out.all_new = all_new ? 1 : 0;
    out.dtype = dtype;
    out.format = format;

    const int64_t slots = cached ? tokens : 0;
    out.table_at = 0;
    out.pages_at = (pages + 1) / 2 * 2;
    out.slots_at = out.pages_at + 2 * pages;
    out.row_tiles_at = (out.slots_at + slots + 3) / 4 * 4;
    if (out.row_tiles_at > capacity)
        return refuse(KVM_EINVAL, "kvm_plan_step: %lld words are too few, kvm_plan_words says how many", (long long)capacity);

    if (cached) {
        std::vector<uint64_t> taken;   // token slots this step writes, one bit each
        taken.assign((size_t)((num_blocks * block_size + 63) / 64), 0);
        int64_t at = 0, slot_at = out.slots_at, row = 0;
        for (int64_t s = 0; s < num_seqs; ++s) {
            const int64_t kv = first_token[s] + new_tokens[s];
            for (int64_t p = 0; p < table_len[s]; ++p) {
                const int64_t block = table[at + p];
                if (block < 0 || block >= num_blocks)
                    return refuse(KVM_ERANGE, "block_table[%lld][%lld] = %lld is outside [0, %lld)", (long long)s,
                                  (long long)p, (long long)block, (long long)num_blocks);
                words[out.table_at + at + p] = (int32_t)block;
                const int64_t done = p * block_size, left = kv - done;
                words[out.pages_at + 2 * (at + p)] = (int32_t)(row + std::min(done, kv));
                words[out.pages_at + 2 * (at + p) + 1] = (int32_t)std::max<int64_t>(0, std::min(left, block_size));
            }
            int64_t page = first_token[s] / block_size, off = first_token[s] % block_size;
            for (int64_t i = 0; i < new_tokens[s]; ++i) {
                const int64_t slot = table[at + page] * block_size + off;
                uint64_t &w = taken[(size_t)(slot >> 6)];
                const uint64_t bit = 1ull << (slot & 63);
                if (w & bit)
                    return refuse(KVM_EDUP, "two tokens of the step go to token %lld of block %lld (sequence %lld)",
                                  (long long)off, (long long)table[at + page], (long long)s);
                w |= bit;
                words[slot_at++] = (int32_t)slot;
                if (++off == block_size) {
                    off = 0;
                    ++page;
                }
            }
            at += table_len[s];
            row += kv;
        }
    }

    // ---- attention work: row tiles, each over the keys its last row may see
    //
    // Sequences of many rows go to the tile kernel (16-bit types; its loads want 16 keys in one block),
    // the others to the row kernel.  (Chunks of 512 behind thousands, 64 heads over 8 of 128, fp16: 350 us over blocks of 16,
    // 1516 us over blocks of 8.)
    auto in_tiles = [&](int64_t s) {
        return dtype != KVM_F32 && new_tokens[s] * group > kFewRows && (!cached || block_size % 16 == 0);
    };
    int64_t most_rows = 0;
    for (int64_t s = 0; s < num_seqs; ++s)
        if (!in_tiles(s)) most_rows = std::max(most_rows, new_tokens[s] * group);
    // Two 16-row tiles share the keys that a wave loads, where the registers hold their accumulators.  The widest sequence decides for
    // the step: 32 sequences of 1500, 32 heads over 8, all of one token or one of them of five, 77 and 125 us in fp32, 37 and 54 us in
    // fp16 over blocks of 8.
    out.row_tiles = most_rows > 16 && head_dim <= 128 ? 2 : 1;

    // few rows: the keys of all (row tile, KV head) pairs in a row, dealt out evenly in units
    std::vector<KvTile> tiles;
    std::vector<KvStart> starts;
    std::vector<KvJoin> joins;
    int64_t units = 0, join_rows = 0, q_start = 0, table_at = 0;
    const int64_t tile_rows = 16 * out.row_tiles;
    for (int64_t s = 0; s < num_seqs; ++s) {
        const int64_t rows = new_tokens[s] * group;
        for (int64_t r = 0; !in_tiles(s) && r < rows; r += tile_rows) {
            const int64_t end = first_token[s] + (std::min(r + tile_rows, rows) - 1) / group + 1;
            tiles.push_back(KvTile{(int32_t)q_start, (int32_t)rows, (int32_t)first_token[s], (int32_t)table_at, (int32_t)r,
                                   (int32_t)end, (int32_t)ceil_div(end, kUnit), 0});
            units += ceil_div(end, kUnit) * num_kv_heads;
        }
        q_start += new_tokens[s];
        if (cached) table_at += table_len[s];
    }
    const int64_t groups = std::min(most_groups(head_dim), units);
    if (groups > 0 && units / groups >= INT32_MAX) return refuse(KVM_EINVAL, "a step of more than 2^31 units of keys a workgroup is not supported");
    {
        size_t tile = 0;
        int64_t head = 0, unit = 0, open = -1;   // open: the group that began the pair at hand and left it unfinished
        for (int64_t w = 0; w < groups; ++w) {
            int64_t left = units / groups + (w < units % groups ? 1 : 0);
            starts.push_back(KvStart{tiles[tile], (int32_t)tile, (int32_t)head, (int32_t)unit, (int32_t)left});
            while (left > 0) {
                const KvTile &t = tiles[tile];
                const int64_t n = std::min<int64_t>(left, t.units - unit);
                if (unit == 0 && n < t.units) open = w;
                left -= n;
                unit += n;
                if (unit < t.units) break;
                if (open >= 0) {
                    const int64_t here = std::min<int64_t>(tile_rows, t.rows - t.row0);
                    joins.push_back(KvJoin{t.q_start, t.row0, (int32_t)here, (int32_t)head, (int32_t)((groups + open) * tile_rows),
                                           (int32_t)((open + 1) * tile_rows), (int32_t)tile_rows, (int32_t)(w - open + 1)});
                    join_rows = std::max(join_rows, here);
                    open = -1;
                }
                unit = 0;
                if (++head == num_kv_heads) {
                    head = 0;
                    ++tile;
                }
            }
        }
    }
    out.row_part_rows = joins.empty() ? 0 : 2 * groups * tile_rows;

    // Many rows: 128-row tiles, their keys cut where that spreads the step over the chip.  Long pieces come first, so that
    // the last workgroups to start are short (chunks among decoding steps, 8 KV heads: 152 us, 164 us by sequence).  With more
    // KV heads than a block has, the tiles of a sequence follow each other for a block's heads at a time instead, so that
    // each die's L2 keeps the one head's K and V that its workgroups read in turn (16 prompts, 32 heads: 367 us, 392 us by length).
    std::vector<KvItem> items;
    std::vector<int64_t> big;
    std::vector<int64_t> row_of((size_t)num_seqs), table_of((size_t)num_seqs);
    int64_t keys = 0, part = 0;
    q_start = table_at = 0;
    for (int64_t s = 0; s < num_seqs; ++s) {
        row_of[(size_t)s] = q_start;
        table_of[(size_t)s] = table_at;
        q_start += new_tokens[s];
        if (cached) table_at += table_len[s];
        if (!in_tiles(s)) continue;
        big.push_back(s);
        for (int64_t r = 0; r < new_tokens[s] * group; r += kTileRows)
            keys += first_token[s] + (std::min(r + kTileRows, new_tokens[s] * group) - 1) / group + 1;
    }
    std::stable_sort(big.begin(), big.end(),
                     [&](int64_t a, int64_t b) { return first_token[a] + new_tokens[a] > first_token[b] + new_tokens[b]; });
    const int64_t all = keys * num_kv_heads, fill = std::min(std::max(ceil_div(all, kTileFill), kShortPiece), kLongPiece);
    const int64_t piece = ceil_div(std::max(ceil_div(all, kTileTarget), fill), kTileStep) * kTileStep;
    std::vector<KvJoin> cut;
    for (int64_t s : big) {
        const int64_t rows = new_tokens[s] * group;
        const size_t begin = items.size();
        for (int64_t r = (rows - 1) / kTileRows * kTileRows; r >= 0; r -= kTileRows) {
            const int64_t here = std::min(kTileRows, rows - r);
            const int64_t end = first_token[s] + (r + here - 1) / group + 1;
            const int64_t cuts = std::max<int64_t>(1, end / piece + (end % piece > piece / 2 ? 1 : 0));
            const int64_t len = ceil_div(ceil_div(end, cuts), kTileStep) * kTileStep;
            const int64_t pieces = ceil_div(end, len);
            for (int64_t p = 0; p < pieces; ++p)
                items.push_back(KvItem{(int32_t)row_of[(size_t)s], (int32_t)rows, (int32_t)first_token[s],
                                       (int32_t)table_of[(size_t)s], (int32_t)r, (int32_t)(p * len),
                                       (int32_t)std::min(end, (p + 1) * len), pieces > 1 ? (int32_t)(part + p * here) : -1, 0, 0, 0, 0});
            if (pieces > 1) {
                cut.push_back(KvJoin{(int32_t)row_of[(size_t)s], (int32_t)r, (int32_t)here, 0, (int32_t)part, (int32_t)(part + here),
                                     (int32_t)here, (int32_t)pieces});
                part += pieces * here;
                join_rows = std::max(join_rows, here);
            }
            if (part * num_kv_heads > kMaxTokens) return refuse(KVM_EINVAL, "a step of more than 2^31 partial rows is not supported");
        }
        const size_t end = items.size();
        for (int64_t head0 = kHeadBlock; head0 < num_kv_heads; head0 += kHeadBlock)
            for (size_t i = begin; i < end; ++i) {
                KvItem it = items[i];
                it.head0 = (int32_t)head0;
                items.push_back(it);
            }
    }
    if (num_kv_heads <= kHeadBlock)
        std::stable_sort(items.begin(), items.end(),
                         [](const KvItem &a, const KvItem &b) { return a.kv_end - a.kv_begin > b.kv_end - b.kv_begin; });
    out.item_part_rows = part;
    out.part_rows = out.row_part_rows + part * num_kv_heads;
    if (out.part_rows > kMaxTokens) return refuse(KVM_EINVAL, "a step of more than 2^31 partial rows is not supported");
    for (const KvJoin &j : cut)
        for (int64_t h = 0; h < num_kv_heads; ++h) {
            KvJoin of_head = j;
            of_head.head = (int32_t)h;
            of_head.part_row += (int32_t)(out.row_part_rows + h * part);
            of_head.next_row += (int32_t)(out.row_part_rows + h * part);
            joins.push_back(of_head);
        }

    out.num_row_tiles = (int64_t)tiles.size();
    out.num_row_groups = groups;
    out.num_tile_items = (int64_t)items.size();
    out.num_joins = (int64_t)joins.size();
    out.join_rows = join_rows;
    int64_t at = out.row_tiles_at;
    auto section = [&](const void *from, size_t bytes) {
        const int64_t here = at;
        at += (int64_t)bytes / 4;
        if (at <= capacity && bytes > 0) memcpy(words + here, from, bytes);
        return here;
    };
    section(tiles.data(), tiles.size() * sizeof(KvTile));
    out.row_starts_at = section(starts.data(), starts.size() * sizeof(KvStart));
    out.tile_items_at = section(items.data(), items.size() * sizeof(KvItem));
    out.joins_at = section(joins.data(), joins.size() * sizeof(KvJoin));
    out.words = at;
    if (out.words > capacity)
        return refuse(KVM_EINVAL, "kvm_plan_step: %lld words are too few, kvm_plan_words says how many", (long long)capacity);
    out.seal = kvm_step_seal(out);
    out.device = -1;
    *step = out;
    return KVM_OK;
} catch (const std::exception &e) {   // out of memory: nothing is thrown through the C interface
    return refuse(KVM_EINVAL, "kvm_plan_step: %s", e.what());
}

int64_t kvm_attention_workspace(const KvmStep *step)
{
    if (!step || step->seal != kvm_step_seal(*step)) return refuse(KVM_EINVAL, "the step is not one kvm_plan_step made");
    return step->part_rows * (step->head_dim + 2) * (int64_t)sizeof(float);
}

}  // extern "C"
