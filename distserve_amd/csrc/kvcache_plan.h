// kvcache_plan.h -- the step plan's work list, as the host writes it and the kernels read it.
#ifndef KVCACHE_PLAN_H
#define KVCACHE_PLAN_H

#include "kvmove.h"

#include <cstddef>

// A piece of attention work for one KV head: rows row0 .. of a sequence over keys [kv_begin, kv_end).
struct KvItem {
    int32_t q_start;    // first token row of the sequence in q and out
    int32_t rows;       // query rows of the sequence for one KV head: new tokens x heads of the group
    int32_t first;      // tokens before the step
    int32_t table_at;   // where the sequence's block table starts
    int32_t row0;
    int32_t kv_begin, kv_end;
    int32_t part_row;   // first partial row of this piece, -1 when the piece is the whole row
};

// Rows whose keys were cut into pieces: piece p's partial rows start at part_row + p * pitch.
struct KvJoin {
    int32_t q_start, row0, rows, part_row, pitch, pieces, pad0, pad1;
};

constexpr int64_t kItemWords = sizeof(KvItem) / 4;
constexpr int64_t kJoinWords = sizeof(KvJoin) / 4;

constexpr int64_t kTargetWorkgroups = 1024;   // four for each of the 256 CUs
constexpr int64_t kPieceStep = 128;           // keys the four waves of a workgroup take in one turn
constexpr int64_t kMinPiece = 256;
constexpr int64_t kFewRows = 32;              // up to here a sequence's rows go to the kernel for few rows
constexpr int64_t kTileRows = 128;            // of a workgroup of the kernel for many rows
constexpr int64_t kTileStep = 64;             // keys of its tiles
constexpr int64_t kMinTilePiece = 512;

uint64_t kvm_step_seal(const KvmStep &s);

#endif  // KVCACHE_PLAN_H
