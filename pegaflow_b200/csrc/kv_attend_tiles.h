// How the tile attention kernel's work is laid out and shared among its CTAs
// (host and device).
//
// An item is a tile of query rows of one sequence for one KV head; its units are
// the key tiles that its rows see. Items in order (sequence, row tile, head) and
// their units within form one line, cut into equal spans, one for each CTA: a
// CTA's span may end inside an item and the next one's begin there. An item that
// lies in several spans is computed in parts and joined afterwards.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kv_ops.h"

namespace pf {

constexpr int kTileRows = 256;  // query rows of an item: two matrix tiles of 128
constexpr int kTileKeys = 128;  // tokens of a unit

struct KvTilePlan {
  uint32_t ctas;
  int32_t page_shift;    // log2 of the block size, -1 if it is no power of two
  uint32_t box_rows;     // tokens of a TMA box, 0: none
  uint32_t reserved;
  uint64_t costs_at;     // byte offsets in the workspace: int64[n_seqs + 1], units in front of each sequence
  uint64_t parts_at;     // float[2 * ctas][dp + 2][kTileRows]: maxima, sums, values
  uint64_t bytes;
};

// Where a CTA's span begins.
struct KvSpan {
  int32_t seq;   // n_seqs: nothing from here on
  int32_t tile;
  int32_t head;
  int32_t unit;
};

__host__ __device__ inline int32_t tile_units(int32_t begin, int32_t end) {
  return end > begin ? (end - begin + kTileKeys - 1) / kTileKeys : 1;  // rows that see nothing are written as well
}

// Units of each CTA's span.
__host__ __device__ inline int64_t span_units(int64_t total, uint32_t ctas) {
  return total > ctas ? (total + ctas - 1) / ctas : 1;
}

// An item that begins at unit `at` of the line: the CTAs that compute it, and
// where each leaves its part (slot 2 c: the first item of its span, 2 c + 1: a
// later one).
struct KvSplit {
  int64_t first;
  int64_t last;
};
__host__ __device__ inline KvSplit item_split(int64_t at, int64_t units, int64_t span) {
  return KvSplit{at / span, (at + units - 1) / span};
}
__host__ __device__ inline int64_t part_slot(int64_t at, int64_t cta, int64_t span) {
  return 2 * cta + (at > cta * span ? 1 : 0);
}

KvTilePlan tile_plan(const KvAttendArgs& k, int num_sms);
cudaError_t launch_attend_tiles(const KvAttendArgs& k, const KvTilePlan& p, cudaStream_t stream);

}  // namespace pf
