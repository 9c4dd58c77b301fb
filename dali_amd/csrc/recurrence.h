// Linear recurrence along sequences and its backward pass.
//   h_t = a_t h_{t-1} + b_t,     DECAY: a = decay, b = x      GATE: a = f = 1 / (1 + exp(-decay)), b = (1 - f) x
//   L_t = dy_t + M_{t+1}, M_t = a_t L_t, behind the last step M = dfinal:     dinitial = M of the first step,
//   DECAY: dx = L, ddecay = L h_{t-1}      GATE: dx = (1 - f) L, ddecay = L (h_{t-1} - x_t) f (1 - f)
//
// A stretch of steps maps the state in front of it to the one behind it: h -> A h + S, A the product of its a_t, S what it makes
// of 0; two stretches one after the other are (A1 A2, A2 S1 + S2).  A workgroup has 128 bytes of channels (16 lanes x 8 bytes) of a
// tile of 256 rows: 32 stretches of 8 steps, one per thread and 8 bytes, held in registers between the two
// times they are needed - for (A, S) of the stretch, and, once the state in front of it is known, for the steps themselves.  The
// states in front come from a scan over the 32 stretches (shuffles inside a wave, the eight waves through LDS) and the state in
// front of the tile.  So memory is read once, in whole lines, however long the dependent chain is.
//
// Rows are one axis over all sequences; a sequence that begins inside a stretch is a step that forgets (R: whatever is in front
// does not count).  Tiles inside one sequence (`interior`) take a path without these tests.
//
// The state in front of a tile is what the tile before leaves behind, which another workgroup has: a chain.  A workgroup says
// what is known as soon as it is known - the product (A, S) of its tile, or the state behind it where that needs nothing from in
// front (a sequence begins in the tile) - and then goes back along the chain, four tiles at a time, adding up products until it
// meets a state.  Every 8th tile says no product, but the state behind it, once it has found the one in front: no tile looks
// further back than that, and which numbers make up a state does not depend on who was first, so neither do its bits.  Tiles are
// given out by a counter in the order of the chain, so a workgroup only ever waits for workgroups that have begun before it and
// waits for none behind them: every wait ends.  Each number is said in one 64-bit word together with a mark that it is there, so
// a number and its mark cannot be seen apart and no fence is needed (a release to the whole card would write back the L2 of an
// XCD); the words are cleared by a launch in front.  With whole sequences in each tile (dense, at most 256 steps) there is no chain.
//
// Of a gate the smaller one of f and 1 - f is computed and applied as such - h + (1 - f)(x - h), or x + f (h - x) - and products of decays
// are held in 64 bits.  With a gate of 0.9999 the rounding of f to 32 bits is an error of 3e-8 in each of ten thousand steps that still
// count, and with constant gates all of one sign; with a gate of 1e-9 that of 1 - f is more than f, and a large state would not go
// away but cancel.
//
// The backward pass runs through the tiles from the last to the first.  It does not use y: the states are computed again in 32
// bits from the one in front of each tile, which the forward pass saves (1/256 of the rows), in the same tile as the L_t: x, decay
// and dy are read once, and with 16-bit types no h is a rounded one.  The states come first; of them the second half needs h_{t-1}
// (gates: h_{t-1} - x_t), which waits in LDS, 64 KB, because registers decide how many workgroups a compute unit holds; for the same
// reason coefficients are computed again from the decays (4 times) rather than kept.  (BackwardChainFirst names the types for which
// registers do not decide, and the chain comes first.)
//
// Measured (gates, bf16, 8 sequences of 4096 steps, 2048 channels; a copy of 1 GiB runs at 5138 GB/s on the same card): forward 118 us
// for 403 MB, 3.4 TB/s; backward 209 us for 671 MB, 3.2 TB/s (with everything in 204 registers and one workgroup per compute unit it
// was 12 % slower).  Decays instead of gates take 7 and 16 % less.  What bounds it is how much is on its way at once, and vector issue
// adds to that.  Holding a gate by the smaller one of f and 1 - f is a quarter more vector instructions than by 1 - f alone, and 5 % of
// the time; without that, a workgroup of the forward pass lived for 10.6 us, of which its loads took 2.4, the scan 3 and the chain 3.3,
// with two per compute unit, and without the chain the pass took 85 us for 110.  Tried and slower: tiles of 64 and of 512 rows; three workgroups
// per compute unit (80 registers); workgroups that stay and load the next tile meanwhile (they hold a place in the chain that they do
// not work on); a chain that all waves listen to; two levels of groups; equal sequences step by step (each tile's predecessor long
// done, but rows far apart in memory at a time); the composition against time in the pass of the other one (256 bytes spilled).
#ifndef DALI_AMD_CSRC_RECURRENCE_H_
#define DALI_AMD_CSRC_RECURRENCE_H_

#include <algorithm>
#include "sequence_common.h"

namespace daliamd {

constexpr int kRecThreads = 512, kRecWaves = kRecThreads / 64;
constexpr int kRecLanes = 16, kRecBytes = 8;          // lanes over channels, bytes of x in each
constexpr int kRecPieces = 64 / kRecLanes;            // stretches per wave
constexpr int kRecSteps = 8;                          // steps per stretch
constexpr int kRecFewSteps = 4;                       // up to so many, a thread goes through a sequence's steps
constexpr int kRecTile = kRecWaves * kRecPieces * kRecSteps;

struct RecKernelArgs {
  daliamdRecurrenceArgs a;
  int tile_rows;                      // kRecTile, or a little less: whole sequences
  int tiles, channel_tiles;
  bool few_steps;                     // a thread goes through a sequence's steps ...
  int first_sequence, sequences;      // ... of these
  bool chained;                       // a tile may need the state behind the one before
  bool x_plain, decay_plain, dy_plain; // rows one distance apart, those of a tile within 32 bits
  uint32_t *ticket;                   // the chain: cleared before each launch, with the words behind it
  uint64_t *words;                    // [tiles][channel_tiles * channels of a tile][kRecWords]
  float *partial;                     // per-channel gradients [tiles][channels]
};
constexpr int kRecGroup = 8;          // tiles from one that says its state to the next
constexpr int kRecWords = 4;          // the state behind the tile; S; A in two halves

// one source file per type of x
template <typename XT> void LaunchRecurrence(hipStream_t s, const RecKernelArgs &p);
template <typename XT> void LaunchRecurrenceBackward(hipStream_t s, const RecKernelArgs &p);

}  // namespace daliamd
#endif  // DALI_AMD_CSRC_RECURRENCE_H_
