// attention_shared_plan.cpp -- which kernel an imq_attention_shared call takes and how its
// keys are split (host code alone).
#include <algorithm>

#include "core_kernels.hpp"
#include "imq_core.h"

namespace imq {
namespace {

constexpr int64_t kPackedBytes = (int64_t)256 << 20;  // of packed documents' sums, at most
constexpr int kStreamStep = kFewWaves * kFewKeys;  // a tile for each wave

// Ranges of at most `chunk` keys (whole steps) over `keys`.
int ranges(int keys, int chunk) { return keys > 0 ? (keys + chunk - 1) / chunk : 0; }

}  // namespace

SharedPlan attention_shared_plan(const AttnArgs& a, const AttnShared& sh, int cus, bool workspace) {
  SharedPlan p{};
  p.kernel = IMQ_SHARED_ROWS;
  const int64_t far = (int64_t)1 << 24;  // elements of a row, as for the own keys
  const int64_t strides = sh.k_row | sh.k_head | sh.v_row | sh.v_head;
  const int64_t own0 = ((int64_t)sh.rows + 2 * kAttnKeys - 1) / (2 * kAttnKeys) * (2 * kAttnKeys);
  // (Rows of values that begin inside the row before: a tile's last would read on past
  // the end of the shared ones.)
  if (strides % 8 != 0 || ((uintptr_t)sh.k | (uintptr_t)sh.v) % 16 != 0 || sh.k_row > far - 128 ||
      sh.v_row > far - 128 || sh.v_row < a.dim || own0 + a.max_k > (1 << 30))
    return p;
  // The walk over both.
  AttnArgs walk = a;
  walk.max_k = (int)own0 + a.max_k;
  p.own0 = (int)own0;
  if (a.max_k == 0) walk.k = walk.v = nullptr;
  p.tiles = attention_plan(walk, cus);
  if (p.tiles.chunk % (2 * kAttnKeys)) {  // ranges of whole pairs of tiles
    const int chunk = p.tiles.chunk + kAttnKeys, splits = ranges(walk.max_k, chunk);
    p.tiles.bytes = p.tiles.bytes / p.tiles.splits * splits;
    p.tiles.chunk = chunk, p.tiles.splits = splits;
  }
  if (p.tiles.kernel == IMQ_ATTENTION_ROWS) return p;
  const int rows = a.max_q * (a.heads / a.kv_heads);
  const int64_t hs = (int64_t)a.n_seq * a.kv_heads;
  p.kernel = IMQ_SHARED_TILES;
  if (p.tiles.kernel == IMQ_ATTENTION_TILES) {
    // Never 256 rows a workgroup, and one sequence after the other where not all workgroups are
    // resident from the start: walks behind a long front are alike, and a sequence's fewer tiles
    // leave no gaps then.  4 x 2048 rows of 32 / 8 heads behind 8192 keys, lengths 2048 / 1265 /
    // 483 / 1749, 828 us against 1027 tile by tile and 1213 with 256 rows; 8 x 2048 of 16 / 4
    // behind 4000 416 / 558 / 609, 32 x 800 behind 2000 553 / 635 / 657; of equal lengths 1175 /
    // 1182 / 1219, 677 / 659 / 681 and 1084 / 1130 / 1137.
    const int64_t hs = (int64_t)a.n_seq * a.kv_heads;
    const int64_t all_rows = (int64_t)a.max_q * (a.heads / a.kv_heads);
    if (p.tiles.tile_rows == 256) p.tiles.tile_rows = 128;
    const int64_t tiles = (all_rows + p.tiles.tile_rows - 1) / p.tiles.tile_rows;
    // (Of few tiles a sequence the empty ones come first, and a CU's share is more even: 61 documents
    // of up to 154 rows behind 3001 keys 119 us against 165.)
    if (p.tiles.splits == 1 && hs * tiles > 2 * cus && tiles >= 8) {
      p.tiles.first = (int)tiles;
      p.tiles.near_hs = a.kv_heads;
    }
    p.bytes = p.tiles.bytes;
    // Packed documents, or batches whose queries lie one sequence behind the other, that leave much of
    // their tiles empty: all rows in one stretch against the shared keys, if the sums' way through memory
    // is worth it.  (Slopes would need every row's sequence there.)  64 sequences of 200 own keys behind 8192,
    // 32 / 8 heads, in tiles and so: of 36 rows 213 and 126 us, 64 214 and 158, 80 235 and 212, but 96 235 and
    // 256, 132 449 and 398, 160 448 and 404; 36 rows of 1000 own keys behind 2048 95 and 92; 32 x 80 behind 1000,
    // where tiles of 64 rows fill the card, 18 and 29.
    const int group = a.heads / a.kv_heads;
    const int64_t line = a.q_offsets ? a.q_rows : a.n_seq * (int64_t)a.max_q;
    const int64_t packed = (line * group + 127) / 128;  // tiles of a key head
    const bool empty = a.q_offsets ? 2 * a.n_seq >= packed
                                   : a.q_seq == a.max_q * a.q_row && p.tiles.tile_rows == 128 &&
                                         all_rows * 8 <= tiles * 128 * 5 && sh.rows >= 2 * (int64_t)a.max_k;
    if (workspace && empty && !a.slopes && p.tiles.splits == 1 && sh.rows >= 512) {
      const int64_t own = hs * ((all_rows + 127) / 128);
      const int64_t blocks = a.kv_heads * packed;
      const int splits = (int)std::max<int64_t>(1, std::min<int64_t>((2 * cus + blocks / 2) / blocks, sh.rows / 512));
      const int chunk = (ranges(sh.rows, splits) + kAttnKeys - 1) / kAttnKeys * kAttnKeys;
      const int d = a.dim > 64 ? 128 : 64;
      const int64_t bytes = ranges(sh.rows, chunk) * blocks * 128 * (d + 2) * (int64_t)sizeof(float);
      if (bytes <= kPackedBytes && std::max(blocks * splits, own) * 256 < ((int64_t)1 << 32)) {
        p.kernel = IMQ_SHARED_PACKED;
        p.s_rows = 128;
        p.s_tiles = (int)packed;
        p.s_chunk = chunk;
        p.s_splits = ranges(sh.rows, chunk);
        p.o_splits = 1;
        p.bytes = (size_t)bytes;
        return p;
      }
    }
    if (p.tiles.splits == 1 || workspace) return p;
  }
  if (p.tiles.kernel == IMQ_ATTENTION_TILES || !workspace) {
    // Unsplit, whatever the rows.
    const int tile_rows = rows > 64 ? 128 : 64;
    const int tiles = (rows + tile_rows - 1) / tile_rows;
    p.tiles = AttnPlan{IMQ_ATTENTION_TILES, tile_rows, 1, tiles, (int)hs, 0, 0};
    p.bytes = 0;
    if (hs * tiles * 512 >= ((int64_t)1 << 32)) p.kernel = IMQ_SHARED_ROWS;
    return p;
  }
  p.kernel = IMQ_SHARED_STREAM;
  const int64_t batch = (int64_t)a.n_seq * rows;
  // 64 rows a workgroup, which halve the reads of the shared keys, where those are more than the
  // L2s keep or the rows many; 32 give a range to more workgroups.  Tokens of 32 / 8 heads behind
  // shared / own keys, 64 rows and 32: 64 behind 8192 / 600 55 and 58 us, behind 65536 / 600 164 and
  // 189, behind 1024 / 256 27.6 and 23.9, 16 behind 4096 / 256 21.6 and 19.4; of 16 / 2 heads behind
  // 8192 / 64 128 tokens 36.5 and 29.3, 512 79 and 82.
  const int64_t tiles64 = (batch + 63) / 64;
  const bool in_l2 = (int64_t)a.kv_heads * sh.rows * a.dim * 4 <= 1 << 24;
  p.s_rows = batch > 32 && !(in_l2 && a.kv_heads * tiles64 * sh.rows < 1 << 19) ? 64 : 32;
  p.s_tiles = (int)((batch + p.s_rows - 1) / p.s_rows);
  // A workgroup a CU: the keys of a range such that all ranges together are as many.  64
  // rows take half as long again as 32.
  const int64_t per = p.s_rows == 64 ? 3 : 2;
  const int64_t work = (int64_t)a.kv_heads * p.s_tiles * sh.rows * per / 2 + hs * a.max_k;
  int64_t chunk = (work + cus - 1) / cus;
  chunk = std::max<int64_t>((chunk + kStreamStep - 1) / kStreamStep * kStreamStep, kStreamStep);
  const int64_t s_chunk = std::max<int64_t>(chunk * 2 / per / kStreamStep * kStreamStep, kStreamStep);
  p.s_splits = ranges(sh.rows, (int)std::min<int64_t>(s_chunk, 1 << 30));
  // Ranges of one length.
  p.s_chunk = (ranges(sh.rows, p.s_splits) + kStreamStep - 1) / kStreamStep * kStreamStep;
  p.s_splits = ranges(sh.rows, p.s_chunk);
  p.o_chunk = (int)std::min<int64_t>(chunk, 1 << 30);
  p.o_splits = ranges(a.max_k, p.o_chunk);
  const int64_t blocks = (int64_t)a.kv_heads * p.s_tiles * p.s_splits + hs * p.o_splits;
  if (std::max(blocks, hs * rows) * 256 >= ((int64_t)1 << 32)) {
    p.kernel = IMQ_SHARED_ROWS;
    return p;
  }
  p.bytes = (size_t)(p.s_splits + p.o_splits) * hs * rows * ((a.dim > 64 ? 128 : 64) + 2) * sizeof(float);
  return p;
}

}  // namespace imq
