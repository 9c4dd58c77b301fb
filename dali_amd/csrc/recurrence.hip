// C entries of the linear recurrence: checks, tiles and workspaces.  recurrence.h says how the kernels work.
#include <algorithm>
#include "recurrence.h"

namespace daliamd {

// Per-channel gradients: the tiles' sums, in a fixed order and in 64 bits, since there are as many as there are rows by the hundred and
// their errors would be of the size of all rows' sum.
constexpr int kRecSumColumns = 16, kRecSumParts = 16;
__global__ __launch_bounds__(kRecSumColumns * kRecSumParts) void RecurrenceChannelSumKernel(RecKernelArgs p) {
  __shared__ double part[kRecSumParts][kRecSumColumns];
  const int column = threadIdx.x % kRecSumColumns, k = threadIdx.x / kRecSumColumns, c = blockIdx.x * kRecSumColumns + column;
  double sum = 0;
  if (c < p.a.channels) {
#pragma unroll 8
    for (int n = k; n < p.tiles; n += kRecSumParts) sum += (double)p.partial[(int64_t)n * p.a.channels + c];
  }
  part[k][column] = sum;
  __syncthreads();
  if (k == 0 && c < p.a.channels) {
    for (int n = 1; n < kRecSumParts; n++) sum += part[n][column];
    StoreElement(p.a.ddecay, c, p.a.decay_dtype, (float)sum);
  }
}

__global__ __launch_bounds__(kRecThreads) void RecurrenceClearKernel(uint4 *words, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kRecThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kRecThreads) words[i] = make_uint4(0, 0, 0, 0);
}

// the initial states, where the call writes the final ones over them
__global__ __launch_bounds__(kRecThreads) void RecurrenceCopyStateKernel(float *to, const float *from, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kRecThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kRecThreads) to[i] = from[i];
}

// ---- launches ------------------------------------------------------------------------------------------------------------
static daliamdResult_t CheckRows(const daliamdSequenceRows &q, const char *what) {
  DALIAMD_REQUIRE(q.rows >= 0 && q.rows <= DALIAMD_SEQUENCE_MAX_ROWS && q.sequences >= 0, DALIAMD_ERROR_OUT_OF_RANGE,
                  "%s: rows must be in [0, %d], sequences not negative", what, (int)DALIAMD_SEQUENCE_MAX_ROWS);
  DALIAMD_REQUIRE(!(q.offsets && q.lengths), DALIAMD_ERROR_INVALID_ARGUMENT, "%s: offsets and lengths exclude each other", what);
  DALIAMD_REQUIRE(!(q.offsets || q.lengths) || q.index_dtype == DALIAMD_INT32 || q.index_dtype == DALIAMD_INT64, DALIAMD_ERROR_UNSUPPORTED,
                  "%s: offsets and lengths must be INT32 or INT64", what);
  DALIAMD_REQUIRE(q.offsets || (q.steps >= 0 && q.steps < ((int64_t)1 << 31) && q.rows == q.steps * q.sequences),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "%s: rows must be sequences * steps", what);
  DALIAMD_REQUIRE(!q.offsets || q.sequences > 0 || q.rows == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "%s: rows without a sequence", what);
  return DALIAMD_SUCCESS;
}

static daliamdResult_t CheckRecurrence(const daliamdRecurrenceArgs *args) {
  DALIAMD_REQUIRE(args, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrence: NULL argument");
  const daliamdRecurrenceArgs &a = *args;
  if (daliamdResult_t r = CheckRows(a.seq, "daliamdRecurrence")) return r;
  DALIAMD_REQUIRE(a.channels >= 1 && a.channels <= DALIAMD_RECURRENCE_MAX_CHANNELS, DALIAMD_ERROR_OUT_OF_RANGE, "daliamdRecurrence: channels must be in [1, %d]", (int)DALIAMD_RECURRENCE_MAX_CHANNELS);
  DALIAMD_REQUIRE(IsSequenceType(a.dtype), DALIAMD_ERROR_UNSUPPORTED, "daliamdRecurrence: x must be FLOAT, FLOAT16 or BFLOAT16");
  DALIAMD_REQUIRE(a.decay_dtype == a.dtype || a.decay_dtype == DALIAMD_FLOAT, DALIAMD_ERROR_UNSUPPORTED,
                  "daliamdRecurrence: decay must have x's type or be FLOAT");
  DALIAMD_REQUIRE(a.form == DALIAMD_RECURRENCE_DECAY || a.form == DALIAMD_RECURRENCE_GATE, DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdRecurrence: unknown form %d", a.form);
  const int channels = kRecLanes * (kRecBytes / ElementSize(a.dtype));
  DALIAMD_REQUIRE((a.seq.rows / kRecTile + 1) * ((a.channels + channels - 1) / channels) <= MaxWorkgroups(kRecThreads), DALIAMD_ERROR_OUT_OF_RANGE,
                  "daliamdRecurrence: more rows and channels than one launch may have");
  return DALIAMD_SUCCESS;
}

// Tiles and workspaces: a function of sizes, types and of whether the states share memory, so that the backward pass finds what the
// forward pass saved, and Setup names what Run takes.
struct RecLayout {
  RecKernelArgs k;
  float *initial_copy;
  size_t chain_bytes, saved_bytes, forward_bytes, backward_bytes;
};
// A few steps per sequence: one thread goes through a sequence's steps.  There is nothing to save then: each tile has whole sequences,
// several of them, so nothing in front of it is the state of one that it has rows of.
static bool FewSteps(const daliamdRecurrenceArgs &a) { return !a.seq.offsets && a.seq.steps > 0 && a.seq.steps <= kRecFewSteps; }
static RecLayout LayOut(const daliamdRecurrenceArgs &a, void *workspace) {
  RecLayout l = {};
  RecKernelArgs &k = l.k;
  k.a = a;
  const daliamdSequenceRows &q = a.seq;
  const int e = ElementSize(a.dtype), d = ElementSize(a.decay_dtype), ch = kRecLanes * (kRecBytes / e);
  k.channel_tiles = (a.channels + ch - 1) / ch;
  // whole sequences in each tile, unless that makes more tiles (of 129 rows instead of 256) than a launch may have
  bool whole = !q.offsets && q.steps > 0 && q.steps <= kRecTile;
  k.tile_rows = whole ? kRecTile / (int)q.steps * (int)q.steps : kRecTile;
  if ((q.rows / k.tile_rows + 1) * k.channel_tiles > MaxWorkgroups(kRecThreads)) whole = false, k.tile_rows = kRecTile;
  k.tiles = (int)std::max<int64_t>(1, (q.rows + k.tile_rows - 1) / k.tile_rows);
  k.chained = !whole && k.tiles > 1;
  auto plain = [&](int64_t row, int64_t seq, int elem) {
    return (q.offsets || q.sequences <= 1 || seq == q.steps * row) && row >= 0 && row <= ((int64_t)1 << 31) / (kRecTile * elem) - kRecTile;
  };
  k.x_plain = plain(a.x_row, a.x_seq, e);
  k.decay_plain = plain(a.decay_row, a.decay_seq, d);
  k.dy_plain = plain(a.dy_row, a.dy_seq, e);
  k.few_steps = whole && FewSteps(a);
  l.saved_bytes = k.few_steps ? 0 : sizeof(float) * (size_t)k.tiles * a.channels;
  uint8_t *at = static_cast<uint8_t *>(workspace);
  size_t used = 0;
  auto take = [&](size_t bytes) {
    uint8_t *p = at + used;
    used += (bytes + 255) & ~(size_t)255;
    return p;
  };
  if (k.chained) {
    k.ticket = reinterpret_cast<uint32_t *>(take(sizeof(uint32_t)));
    k.words = reinterpret_cast<uint64_t *>(take(sizeof(uint64_t) * kRecWords * (size_t)k.tiles * k.channel_tiles * ch));
    l.chain_bytes = used;
  }
  const size_t states = sizeof(float) * (size_t)q.sequences * a.channels;
  const uint8_t *initial = reinterpret_cast<const uint8_t *>(a.initial), *final_state = reinterpret_cast<const uint8_t *>(a.final_state);
  l.forward_bytes = used;
  // Initial states are read while others' final ones are written; only where a thread has all of a state, and writes it where it read it,
  // that is no matter.
  const bool overlap = initial && final_state && initial < final_state + states && final_state < initial + states;
  if (overlap && !(k.few_steps && initial == final_state)) {
    const size_t before = used;
    l.initial_copy = reinterpret_cast<float *>(take(states));
    l.forward_bytes = used;
    used = before;
  }
  if (a.per_channel) k.partial = reinterpret_cast<float *>(take(sizeof(float) * (size_t)k.tiles * a.channels));
  l.backward_bytes = used;
  return l;
}

static void ClearChain(hipStream_t s, const RecLayout &l) {
  if (!l.chain_bytes || l.k.few_steps) return;
  const int64_t n = l.chain_bytes / sizeof(uint4);
  KernelTimer timer("RecurrenceClearKernel", s);
  hipLaunchKernelGGL(RecurrenceClearKernel, dim3((unsigned)std::min<int64_t>((n + kRecThreads - 1) / kRecThreads, 1024)), dim3(kRecThreads), 0, s,
                     reinterpret_cast<uint4 *>(l.k.ticket), n);
}

}  // namespace daliamd

extern "C" {

daliamdResult_t daliamdRecurrenceSetup(const daliamdRecurrenceArgs *args, daliamdRecurrencePlan *plan) {
  using namespace daliamd;
  DALIAMD_REQUIRE(plan, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceSetup: NULL argument");
  if (daliamdResult_t r = CheckRecurrence(args)) return r;
  const RecLayout l = LayOut(*args, nullptr);
  plan->saved_bytes = l.saved_bytes;
  plan->forward_workspace_bytes = l.forward_bytes;
  plan->backward_workspace_bytes = l.backward_bytes;
  return DALIAMD_SUCCESS;
}

daliamdResult_t daliamdRecurrenceRun(daliamdStream_t stream, const daliamdRecurrenceArgs *args, void *workspace, size_t workspace_bytes) {
  using namespace daliamd;
  if (daliamdResult_t r = CheckRecurrence(args)) return r;
  const daliamdSequenceRows &q = args->seq;
  RecLayout l = LayOut(*args, workspace);
  DALIAMD_REQUIRE(q.rows == 0 || (args->x && args->decay && args->y), DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceRun: NULL tensor");
  DALIAMD_REQUIRE(workspace_bytes >= l.forward_bytes && (workspace || !l.forward_bytes), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdRecurrenceRun: the workspace is too small");
  DALIAMD_REQUIRE((uintptr_t)workspace % 16 == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceRun: the workspace must start at a multiple of 16 bytes");
  if (!q.sequences) return DALIAMD_SUCCESS;
  hipStream_t s = (hipStream_t)stream;
  if (l.initial_copy) {
    const int64_t n = (int64_t)q.sequences * args->channels;
    KernelTimer timer("RecurrenceCopyStateKernel", s);
    hipLaunchKernelGGL(RecurrenceCopyStateKernel, dim3((unsigned)std::min<int64_t>((n + kRecThreads - 1) / kRecThreads, 4096)), dim3(kRecThreads), 0, s,
                       l.initial_copy, args->initial, n);
    l.k.a.initial = l.initial_copy;
  }
  ClearChain(s, l);
  if (args->dtype == DALIAMD_FLOAT) LaunchRecurrence<float>(s, l.k);
  else if (args->dtype == DALIAMD_FLOAT16) LaunchRecurrence<F16>(s, l.k);
  else LaunchRecurrence<Bf16>(s, l.k);
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

daliamdResult_t daliamdRecurrenceBackwardRun(daliamdStream_t stream, const daliamdRecurrenceArgs *args, void *workspace,
                                             size_t workspace_bytes) {
  using namespace daliamd;
  if (daliamdResult_t r = CheckRecurrence(args)) return r;
  const daliamdSequenceRows &q = args->seq;
  RecLayout l = LayOut(*args, workspace);
  DALIAMD_REQUIRE((args->ddecay || (q.rows == 0 && !args->per_channel)) && (q.rows == 0 || (args->x && args->decay && args->dx && (args->saved || !l.saved_bytes))),
                  DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceBackwardRun: NULL tensor");
  DALIAMD_REQUIRE(workspace_bytes >= l.backward_bytes && (workspace || !l.backward_bytes), DALIAMD_ERROR_INVALID_ARGUMENT,
                  "daliamdRecurrenceBackwardRun: the workspace is too small");
  DALIAMD_REQUIRE((uintptr_t)workspace % 16 == 0, DALIAMD_ERROR_INVALID_ARGUMENT, "daliamdRecurrenceBackwardRun: the workspace must start at a multiple of 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  l.k.few_steps = false;
  if (!l.saved_bytes) l.k.a.saved = nullptr;
  ClearChain(s, l);
  if (args->dtype == DALIAMD_FLOAT) LaunchRecurrenceBackward<float>(s, l.k);
  else if (args->dtype == DALIAMD_FLOAT16) LaunchRecurrenceBackward<F16>(s, l.k);
  else LaunchRecurrenceBackward<Bf16>(s, l.k);
  if (args->per_channel) {
    KernelTimer timer("RecurrenceChannelSumKernel", s);
    hipLaunchKernelGGL(RecurrenceChannelSumKernel, dim3((args->channels + kRecSumColumns - 1) / kRecSumColumns), dim3(kRecSumColumns * kRecSumParts), 0, s, l.k);
  }
  DALIAMD_HIP_CHECK(hipGetLastError());
  return DALIAMD_SUCCESS;
}

}  // extern "C"
