// Linear recurrence along sequences and its backward pass.
//   h_t = a_t h_{t-1} + b_t,     DECAY: a = decay, b = x      GATE: a = f = 1 / (1 + exp(-decay)), b = (1 - f) x
//   L_t = dy_t + M_{t+1}, M_t = a_t L_t, behind the last step M = dfinal:     dinitial = M of the first step,
//   DECAY: dx = L, ddecay = L h_{t-1}      GATE: dx = (1 - f) L, ddecay = L (h_{t-1} - x_t) f (1 - f)
//
// A stretch of steps maps the state in front of it to the one behind it: h -> A h + S, A the product of its a_t, S what it makes
// of 0; two stretches one after the other are (A1 A2, A2 S1 + S2).  A workgroup has 128 bytes of channels (8 lanes x 16 bytes) and
// goes through the rows in tiles of 256: 32 stretches of 8 steps, one per thread and 16 bytes, held in registers between the two
// times they are needed - for (A, S) of the stretch, and, once the state in front of it is known, for the steps themselves.  The
// states in front come from a scan over the 32 stretches (shuffles inside a wave, the four waves through LDS) and the state behind
// the tile before, which stays in registers.  So memory is read once, in whole lines, however long the dependent chain is.
//
// Rows are one axis over all sequences; a sequence that begins inside a stretch is a step that forgets (R: whatever is in front
// does not count).  Tiles inside one sequence (`interior`) take a path without these tests.
//
// 1 - f is computed and applied as such (h += (1 - f)(x - h)), and products of decays are held in 64 bits: with a gate of 0.9999
// the rounding of f to 32 bits is an error of 3e-8 in each of ten thousand steps that still count, and with constant gates all
// of one sign.
//
// Where sequences times channel groups are too few workgroups to fill the card, or the host does not know where sequences begin,
// the rows are cut into chunks of whole tiles: RecurrenceChunkKernel finds (A, S, R) of each, and the kernels then start from the
// scan over the chunks in front.  That reads the inputs twice.
//
// The backward pass runs through the tiles from the last to the first.  It does not use y: the states are computed again in 32
// bits from the one in front of each tile, which the forward pass saves (1/256 of the rows), in the same tile as the L_t: x, decay
// and dy are read once, and with 16-bit types no h is a rounded one.
#ifndef DALI_AMD_CSRC_RECURRENCE_H_
#define DALI_AMD_CSRC_RECURRENCE_H_

#include "sequence_common.h"

namespace daliamd {

constexpr int kRecThreads = 256, kRecWaves = kRecThreads / 64;
constexpr int kRecLanes = 8;                          // lanes over channels
constexpr int kRecPieces = 64 / kRecLanes;            // stretches per wave
constexpr int kRecSteps = 8;                          // steps per stretch
constexpr int kRecFewSteps = 4;                       // up to so many, a thread goes through a sequence's steps
constexpr int kRecTile = kRecWaves * kRecPieces * kRecSteps;

struct RecKernelArgs {
  daliamdRecurrenceArgs a;
  int64_t chunk_rows;
  int chunks, tiles, channel_tiles;   // tiles: per chunk
  bool few_steps;                     // a thread goes through a sequence's steps
  bool joined;                        // chunks are parts of sequences: their products below are there
  bool x_wide, decay_wide, dy_wide, out_wide, decay_out_wide;
  double *chunk_a;                    // [chunks][channels]
  float *chunk_s;                     // [chunks][channels]
  int *chunk_r;                       // [chunks][channel_tiles]
  float *partial;                     // per-channel gradients [chunks][channels]
};

// one source file per type of x
template <typename XT> void LaunchRecurrence(hipStream_t s, const RecKernelArgs &p);
template <typename XT> void LaunchRecurrenceBackward(hipStream_t s, const RecKernelArgs &p);

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_RECURRENCE_H_
