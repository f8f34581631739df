// Where the attention kernels of the 4-bit cache look, as plain arithmetic without a type of the GPU's: constexpr functions, which
// device code calls as they are and a host compiler can check up to the lengths' limit.
#ifndef QF_KV4_PLACES_H
#define QF_KV4_PLACES_H

#include <stdint.h>

#include "qf_kv4.h"

namespace qfk {

constexpr int kTile = QF_KV4_TILE;  // positions of a cache record
constexpr int kStep = 2 * kTile;    // positions of a step of attn_split_kernel
constexpr int kStage = 4 * kTile;   // positions of a stage of attn_tile_kernel

// The position of record `lane` (0 .. 63) from stage `stage` on, or the last record's. A kernel looks up to two stages past its
// last one ahead: of 2^31 - 64 positions that is position 2^31, which 31 bits do not hold.
constexpr int stage_record(int stage, int lane, int last_tile) {
  const uint32_t pos = (uint32_t)stage * kStage + (uint32_t)lane * kTile;
  return pos < (uint32_t)last_tile ? (int)pos : last_tile;
}

// Steps of a chunk where `workers` chunks share `total` steps, at most a sequence's (65 535 sequences of them on one worker are 2^42,
// more than 32 bits hold).
constexpr uint32_t kMostSteps = 1u << 26;
constexpr uint32_t chunk_steps(uint64_t total, uint32_t workers) {
  const uint64_t steps = total / workers + 1;
  return steps < kMostSteps ? (uint32_t)steps : kMostSteps;
}

}  // namespace qfk

#endif
