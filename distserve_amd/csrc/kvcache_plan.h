// kvcache_plan.h -- the step plan's work list, as the host writes it and the kernels read it.
#ifndef KVCACHE_PLAN_H
#define KVCACHE_PLAN_H

#include "kvmove.h"

#include <cstddef>

// A row tile of a sequence, for the kernel for few rows: the same for every KV head.
struct KvTile {
    int32_t q_start;    // first token row of the sequence in q and out
    int32_t rows;       // query rows of the sequence for one KV head: new tokens x heads of the group
    int32_t first;      // tokens before the step
    int32_t table_at;   // where the sequence's block table starts
    int32_t row0;
    int32_t kv_end;     // keys that the tile's last row may see
    int32_t units, pad; // of kUnit keys
};

// Where a workgroup of the kernel for few rows starts: the units of all (tile, KV head) pairs in a row are
// dealt out evenly, so that every workgroup has the same amount to read.
struct KvStart {
    KvTile first;       // the tile it starts with
    int32_t tile, head, unit, units;
};

// A piece of attention work for the kernel for many rows: rows row0 .. over keys [kv_begin, kv_end), for KV heads
// head0 .. head0 + kHeadBlock - 1 (those that exist).
struct KvItem {
    int32_t q_start, rows, first, table_at, row0;   // as above
    int32_t kv_begin, kv_end;
    int32_t part_row;   // first partial row of this piece for KV head 0, -1 when the piece is the whole row
    int32_t head0, pad0, pad1, pad2;
};

// Rows of one KV head whose keys were cut into pieces: partial rows start at part_row, then at next_row + i * pitch.
struct KvJoin {
    int32_t q_start, row0, rows, head, part_row, next_row, pitch, pieces;
};

constexpr int64_t kTileWords = sizeof(KvTile) / 4;
constexpr int64_t kStartWords = sizeof(KvStart) / 4;
constexpr int64_t kItemWords = sizeof(KvItem) / 4;
constexpr int64_t kJoinWords = sizeof(KvJoin) / 4;

constexpr int64_t kUnit = 128;                // keys the four waves of a workgroup for few rows take in one turn
constexpr int64_t kCus = 256;
// Up to here a sequence's rows go to the kernel for few rows.  16 sequences of 2048, 8 KV heads of 128, fp16, in us: 16 rows 31.6
// there, 42.3 in the kernel for many; 24 rows 55.4 and 42.6; 32 heads of 1000 keys, 24 rows 80.7 and 56.1.
constexpr int64_t kFewRows = 16;
constexpr int64_t kTileRows = 128;            // of a workgroup of the kernel for many rows
constexpr int64_t kTileStep = 64;             // keys of its tiles
// How long the pieces are that it is cut into: a step fills the chip with some 384 workgroups, by pieces of 256 keys at
// least, and then with up to 1024, by pieces of 1024 at least: more pieces even the load out, but each writes its rows in 32
// bits and the join reads them.  One piece length for all would be (us, 512 and 1024 keys) 21.4 and 30.8 for a chunk of 64 behind
// 4000, 67.6 and 55.5 for one of 256 behind 8000; 512, 768 or 1536 workgroups instead of 1024: 163, 160, 161 for 152
// (two chunks among decoding steps).
constexpr int64_t kTileTarget = 1024;
constexpr int64_t kTileFill = 384;
constexpr int64_t kShortPiece = 256;
constexpr int64_t kLongPiece = 1024;
constexpr int64_t kHeadBlock = 8;             // KV heads side by side: one for each of the chip's eight dies, which have an L2 each

uint64_t kvm_step_seal(const KvmStep &s);

#endif  // KVCACHE_PLAN_H
