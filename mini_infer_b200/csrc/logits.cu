// What requests ask of their logits, and the token histories that it takes.
//
//   z = logit                                    of token v in the row of a request
//   z = z > 0 ? z / r : z r                      where the request's history holds v (prompt or generated)
//   z = z - f c - p                              where c > 0, c the times that v was generated
//   z = z + b                                    for every bias (v, b) that the request gives
//   z = -inf                                     where the request's mask has no bit for v
//
// in this order, every operation rounded to fp32 on its own.  A history is a row of `seen` (bit v % 32 of word v / 32)
// and a row of `counts` (int32 a token).
#include "common.cuh"

MI_DEFINE_ERROR_API()

#define ADJUST_THREADS 256
#define ADJUST_COLS 8192      // columns of a row that a block takes (a multiple of 32)

struct AdjustArgs {
  const float* logits;
  float* out;
  long long ld_in, ld_out;
  int V, words;
  const int* slots;                  // row of the histories, or negative: none
  const uint32_t* seen;
  const int* counts;
  int n_slots;
  const float *repetition, *presence, *frequency;
  const int *bias_starts, *bias_ids;
  const float* bias_values;
  int n_bias;
  const uint32_t* masks;
  const int* mask_rows;
  int n_masks;
};

__global__ void __launch_bounds__(ADJUST_THREADS) adjust_logits_kernel(const AdjustArgs a) {
  mi_pdl_enter();   // the logits and the histories come from the kernels before this one
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* in = a.logits + (size_t)row * a.ld_in;
  float* out = a.out + (size_t)row * a.ld_out;
  const bool in_place = in == out;
  const int begin = blockIdx.x * ADJUST_COLS, end = min(a.V, begin + ADJUST_COLS);

  const int slot = a.seen ? (a.slots ? a.slots[row] : row) : -1;
  const bool known = slot >= 0 && slot < a.n_slots;
  const uint32_t* seen = known ? a.seen + (size_t)slot * a.words : nullptr;
  const int* counts = known && a.counts ? a.counts + (size_t)slot * a.V : nullptr;
  const float rep = known && a.repetition ? a.repetition[row] : 1.f;
  const float pres = known && a.presence ? a.presence[row] : 0.f;
  const float freq = known && a.frequency ? a.frequency[row] : 0.f;
  const int mrow = a.masks ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
  const uint32_t* mask = mrow >= 0 && mrow < a.n_masks ? a.masks + (size_t)mrow * a.words : nullptr;

  for (int c0 = begin + warp * 32; c0 < end; c0 += ADJUST_THREADS) {
    const int v = c0 + lane;
    if (v >= end) break;
    const uint32_t told = seen ? seen[c0 >> 5] : 0u, open = mask ? mask[c0 >> 5] : ~0u;
    const bool here = (told >> lane) & 1u, shut = !((open >> lane) & 1u);
    if (in_place && !here && !shut) continue;
    float z = in[v];
    if (here) {
      z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
      const int c = counts ? counts[v] : 0;
      if (c > 0) z = __fsub_rn(__fsub_rn(z, __fmul_rn(freq, (float)c)), pres);
    }
    out[v] = shut ? -INFINITY : z;
  }
  if (!a.bias_starts) return;
  __syncthreads();
  if (warp) return;
  // One warp adds the biases of the block's columns, in the order of the list: of equal ids within 32 entries the first
  // one's lane adds all, so that every sum has one order.
  const int first = max(0, a.bias_starts[row]), last = min(a.n_bias, a.bias_starts[row + 1]);
  for (int j0 = first; j0 < last; j0 += 32) {
    const int j = j0 + lane;
    int v = -1;
    float b = 0.f;
    if (j < last) {
      v = a.bias_ids[j];
      b = a.bias_values[j];
    }
    const bool mine = v >= begin && v < end && (!mask || ((mask[v >> 5] >> (v & 31)) & 1u));
    const unsigned same = __match_any_sync(0xffffffffu, mine ? v : -1 - lane);
    const bool leads = mine && lane == __ffs(same) - 1;
    float z = leads ? out[v] : 0.f;
    unsigned any = __ballot_sync(0xffffffffu, mine);
    while (any) {
      const int from = __ffs(any) - 1;
      any &= any - 1;
      const float add = __shfl_sync(0xffffffffu, b, from);
      if (leads && ((same >> from) & 1u)) z = __fadd_rn(z, add);
    }
    if (leads) out[v] = z;
    __syncwarp();
  }
}

extern "C" int mi_adjust_logits(const float* logits, long long ld_in, float* out, long long ld_out, int B, int V,
                                const int* slots, const uint32_t* seen, const int* counts, int n_slots,
                                const float* repetition, const float* presence, const float* frequency,
                                const int* bias_starts, const int* bias_ids, const float* bias_values, int n_bias,
                                const uint32_t* masks, const int* mask_rows, int n_masks, cudaStream_t stream) {
  if (B <= 0 || V <= 0) return 0;
  if (B > 65535) MI_REFUSE("adjust_logits: %d rows, at most 65535", B);
  if (V > 0x7fffffff - ADJUST_COLS) MI_REFUSE("adjust_logits: vocabulary %d", V);
  AdjustArgs a = {logits, out, ld_in, ld_out, V, (int)(((long long)V + 31) / 32), slots, seen, counts, n_slots, repetition,
                  presence, frequency, bias_starts, bias_ids, bias_values, n_bias, masks, mask_rows, n_masks};
  MI_LAUNCH((adjust_logits_kernel), dim3((V + ADJUST_COLS - 1) / ADJUST_COLS, B), ADJUST_THREADS, 0, stream, a);
  MI_RETURN_LAUNCH_STATUS();
}

// ---------------------------------------------------------------------------------------------- histories

#define RECORD_THREADS 256
#define RECORD_COLS 8192

// Tokens [first, last) are the request's (without `starts`: one token each), those from `made` on are generated ones.
__device__ __forceinline__ void tokens_of(int req, const int* starts, int n_tokens, const int* n_prompt, int& first, int& last,
                                          long long& made) {
  const int from = starts ? starts[req] : req;
  first = max(0, from);
  last = min(n_tokens, starts ? starts[req + 1] : req + 1);
  made = n_prompt ? (long long)from + n_prompt[req] : from;
}

// A history written anew: the block counts the request's tokens within its stretch of the vocabulary in shared memory
// (whole numbers: their order does not matter) and writes the stretch once.
__global__ void __launch_bounds__(RECORD_THREADS)
record_fresh_kernel(int* counts, uint32_t* seen, int n_slots, int V, int words, const int* slots, const int* starts,
                    const int* tokens, int n_tokens, const int* n_prompt) {
  mi_pdl_enter();
  __shared__ int tally[RECORD_COLS];
  __shared__ uint32_t bits[RECORD_COLS / 32];
  const int req = blockIdx.y, tid = threadIdx.x;
  const int begin = blockIdx.x * RECORD_COLS, end = min(V, begin + RECORD_COLS);
  const int slot = slots ? slots[req] : req;
  if (slot < 0 || slot >= n_slots) return;
  for (int i = tid; i < RECORD_COLS; i += RECORD_THREADS) tally[i] = 0;
  for (int i = tid; i < RECORD_COLS / 32; i += RECORD_THREADS) bits[i] = 0u;
  __syncthreads();
  int first, last;
  long long made;
  tokens_of(req, starts, n_tokens, n_prompt, first, last, made);
  for (int i = first + tid; i < last; i += RECORD_THREADS) {
    const int v = tokens[i];
    if (v < begin || v >= end) continue;
    atomicOr(&bits[(v - begin) >> 5], 1u << (v & 31));
    if (i >= made) atomicAdd(&tally[v - begin], 1);
  }
  __syncthreads();
  int* c = counts + (size_t)slot * V;
  for (int v = begin + tid; v < end; v += RECORD_THREADS) c[v] = tally[v - begin];
  uint32_t* s = seen + (size_t)slot * words;
  const int wend = min(words, (begin + RECORD_COLS) / 32);
  for (int w = begin / 32 + tid; w < wend; w += RECORD_THREADS) s[w] = bits[w - begin / 32];
}

// Tokens added to what a history holds.
__global__ void __launch_bounds__(RECORD_THREADS)
record_more_kernel(int* counts, uint32_t* seen, int n_slots, int V, int words, const int* slots, const int* starts,
                   const int* tokens, int n_tokens, const int* n_prompt) {
  mi_pdl_enter();
  const int req = blockIdx.x;
  const int slot = slots ? slots[req] : req;
  if (slot < 0 || slot >= n_slots) return;
  int first, last;
  long long made;
  tokens_of(req, starts, n_tokens, n_prompt, first, last, made);
  for (int i = first + threadIdx.x; i < last; i += RECORD_THREADS) {
    const int v = tokens[i];
    if (v < 0 || v >= V) continue;
    atomicOr(&seen[(size_t)slot * words + (v >> 5)], 1u << (v & 31));
    if (i >= made) atomicAdd(&counts[(size_t)slot * V + v], 1);
  }
}

extern "C" int mi_record_tokens(int* counts, uint32_t* seen, int n_slots, int V, const int* slots, const int* starts,
                                const int* tokens, int n_tokens, const int* n_prompt, int B, int fresh,
                                cudaStream_t stream) {
  if (B <= 0 || V <= 0) return 0;
  if (B > 65535) MI_REFUSE("record_tokens: %d requests, at most 65535", B);
  if (V > 0x7fffffff - RECORD_COLS) MI_REFUSE("record_tokens: vocabulary %d", V);
  const int words = (int)(((long long)V + 31) / 32);
  if (fresh)
    MI_LAUNCH((record_fresh_kernel), dim3((V + RECORD_COLS - 1) / RECORD_COLS, B), RECORD_THREADS, 0, stream, counts, seen,
              n_slots, V, words, slots, starts, tokens, n_tokens, n_prompt);
  else
    MI_LAUNCH((record_more_kernel), B, RECORD_THREADS, 0, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt);
  MI_RETURN_LAUNCH_STATUS();
}
