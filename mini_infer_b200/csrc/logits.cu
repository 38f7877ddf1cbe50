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
#define ADJUST_GROUPS 4       // groups of 4 columns that a thread has under way at once
#define ADJUST_COLS (ADJUST_THREADS * ADJUST_GROUPS * 4)

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

// The bits of columns c .. c + 3 of a row of bits.
__device__ __forceinline__ uint32_t four_bits(const uint32_t* row, int c, int words) {
  const int w = c >> 5;
  return __funnelshift_r(row[w], row[min(w + 1, words - 1)], c & 31) & 15u;
}

// A block takes ADJUST_COLS columns of one row, a thread four groups of four columns: all its loads are under way before the
// first is looked at, and a row that starts off a 16-byte boundary is taken from its first boundary on (the up to three columns
// in front are a group of their own).  In place, a group of which nothing changes is neither read nor written.
template <bool IN_PLACE>
__global__ void __launch_bounds__(ADJUST_THREADS) adjust_logits_kernel(const AdjustArgs a) {
  mi_pdl_enter();   // the logits and the histories come from the kernels before this one
  __shared__ float bias_at[ADJUST_COLS + 4];
  __shared__ uint32_t biased[ADJUST_COLS / 32 + 1];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const float* in = a.logits + (size_t)row * a.ld_in;
  float* out = a.out + (size_t)row * a.ld_out;
  // columns before the first 16-byte boundary, and this block's columns: [begin, end), the first block's from 0 on
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / 4;
  const int start = blockIdx.x * ADJUST_COLS + head;
  const int begin = blockIdx.x ? start : 0, end = min(a.V, start + ADJUST_COLS);
  const bool vec_out = (reinterpret_cast<uintptr_t>(out + head) & 15) == 0;

  float4 z[ADJUST_GROUPS];
  if (!IN_PLACE) {
#pragma unroll
    for (int j = 0; j < ADJUST_GROUPS; ++j) {
      const int c = start + (j * ADJUST_THREADS + tid) * 4;
      if (c + 4 <= end) z[j] = *reinterpret_cast<const float4*>(in + c);
    }
  }
  const int slot = a.seen ? (a.slots ? a.slots[row] : row) : -1;
  const int mrow = a.masks ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
  const bool known = slot >= 0 && slot < a.n_slots, masked = mrow >= 0 && mrow < a.n_masks;
  const uint32_t* seen = a.seen + (size_t)(known ? slot : 0) * a.words;
  const uint32_t* mask = a.masks + (size_t)(masked ? mrow : 0) * a.words;
  uint32_t told[ADJUST_GROUPS], shut[ADJUST_GROUPS];
#pragma unroll
  for (int j = 0; j < ADJUST_GROUPS; ++j) {
    const int c = start + (j * ADJUST_THREADS + tid) * 4;
    told[j] = known && c < end ? four_bits(seen, c, a.words) : 0u;
    shut[j] = masked && c < end ? ~four_bits(mask, c, a.words) & 15u : 0u;
  }
  const float rep = known && a.repetition ? a.repetition[row] : 1.f;
  const float pres = known && a.presence ? a.presence[row] : 0.f;
  const float freq = known && a.frequency ? a.frequency[row] : 0.f;
  const int* counts = known && a.counts ? a.counts + (size_t)slot * a.V : nullptr;

  // The biases of this block's columns into shared memory, a bit for each column that has one.  One warp adds them in the
  // order of the list: of equal ids within 32 entries the first one's lane adds all, so that every sum has one order.
  const bool biases = a.bias_starts != nullptr;
  if (biases) {
    for (int i = tid; i < ADJUST_COLS / 32 + 1; i += ADJUST_THREADS) biased[i] = 0u;
    __syncthreads();
    if (tid < 32) {
      const int first = max(0, a.bias_starts[row]), last = min(a.n_bias, a.bias_starts[row + 1]);
      for (int j0 = first; j0 < last; j0 += 128) {
        int ids[4];
        float values[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + 32 * u + lane;
          ids[u] = j < last ? a.bias_ids[j] : -1;
          values[u] = j < last ? a.bias_values[j] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool mine = ids[u] >= begin && ids[u] < end;
          unsigned any = __ballot_sync(0xffffffffu, mine);
          if (!any) continue;
          const unsigned same = __match_any_sync(0xffffffffu, mine ? ids[u] : -1 - lane);
          const bool leads = mine && lane == __ffs(same) - 1;
          const int at = ids[u] - begin;
          bool there = leads && ((biased[at >> 5] >> (at & 31)) & 1u);
          float sum = there ? bias_at[at] : 0.f;
          while (any) {
            const int from = __ffs(any) - 1;
            any &= any - 1;
            const float add = __shfl_sync(0xffffffffu, values[u], from);
            if (leads && ((same >> from) & 1u)) {
              sum = there ? __fadd_rn(sum, add) : add;
              there = true;
            }
          }
          __syncwarp();
          if (leads) {
            bias_at[at] = sum;
            atomicOr(&biased[at >> 5], 1u << (at & 31));
          }
          __syncwarp();
        }
      }
    }
    __syncthreads();
  }

  const auto one = [&](float v, int c, bool here, bool closed, bool more) {
    if (here) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      const int n = counts ? counts[c] : 0;
      if (n > 0) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)n)), pres);
    }
    if (more) v = __fadd_rn(v, bias_at[c - begin]);
    return closed ? -INFINITY : v;
  };
#pragma unroll
  for (int j = 0; j < ADJUST_GROUPS; ++j) {
    const int c = start + (j * ADJUST_THREADS + tid) * 4;
    if (c >= end) break;
    uint32_t more = 0u;
    if (biases) {
      const int w = (c - begin) >> 5;
      more = __funnelshift_r(biased[w], biased[min(w + 1, ADJUST_COLS / 32)], (c - begin) & 31) & 15u;
    }
    const uint32_t changed = told[j] | shut[j] | more;
    if (IN_PLACE && !changed) continue;
    if (c + 4 <= end) {
      if (IN_PLACE) z[j] = *reinterpret_cast<const float4*>(in + c);
      if (changed) {
        z[j].x = one(z[j].x, c, told[j] & 1u, shut[j] & 1u, more & 1u);
        z[j].y = one(z[j].y, c + 1, told[j] & 2u, shut[j] & 2u, more & 2u);
        z[j].z = one(z[j].z, c + 2, told[j] & 4u, shut[j] & 4u, more & 4u);
        z[j].w = one(z[j].w, c + 3, told[j] & 8u, shut[j] & 8u, more & 8u);
      }
      if (vec_out) {
        *reinterpret_cast<float4*>(out + c) = z[j];
      } else {
        out[c] = z[j].x; out[c + 1] = z[j].y; out[c + 2] = z[j].z; out[c + 3] = z[j].w;
      }
    } else {
      for (int i = 0; c + i < end; ++i) out[c + i] = one(in[c + i], c + i, (told[j] >> i) & 1u, (shut[j] >> i) & 1u, (more >> i) & 1u);
    }
  }
  if (blockIdx.x == 0 && tid < min(head, a.V)) {          // the columns before the boundary
    const uint32_t here = known ? (seen[0] >> tid) & 1u : 0u, closed = masked ? ~(mask[0] >> tid) & 1u : 0u;
    const uint32_t more = biases ? (biased[0] >> tid) & 1u : 0u;
    if (!IN_PLACE || (here | closed | more)) out[tid] = one(in[tid], tid, here, closed, more);
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
  const bool in_place = out == logits;
  AdjustArgs a = {logits, out, ld_in, ld_out, V, (int)(((long long)V + 31) / 32), slots, seen, counts, n_slots, repetition,
                  presence, frequency, bias_starts, bias_ids, bias_values, n_bias, masks, mask_rows, n_masks};
  // (a row whose first columns lie before a boundary may need no more blocks for it: the first block's stretch is the longer)
  const dim3 grid((V + ADJUST_COLS - 1) / ADJUST_COLS, B);
  if (in_place)
    MI_LAUNCH((adjust_logits_kernel<true>), grid, ADJUST_THREADS, 0, stream, a);
  else
    MI_LAUNCH((adjust_logits_kernel<false>), grid, ADJUST_THREADS, 0, stream, a);
  MI_RETURN_LAUNCH_STATUS();
}

// ---------------------------------------------------------------------------------------------- histories

#define RECORD_THREADS 512

// Tokens [first, last) are the request's (without `starts`: one token each), those from `made` on are generated ones.
__device__ __forceinline__ void tokens_of(int req, const int* starts, int n_tokens, const int* n_prompt, int& first, int& last,
                                          long long& made) {
  const int from = starts ? starts[req] : req;
  first = max(0, from);
  last = min(n_tokens, starts ? starts[req + 1] : req + 1);
  made = n_prompt ? (long long)from + n_prompt[req] : from;
}

// A history written anew: the block counts the request's tokens within its stretch of the vocabulary in shared memory
// (whole numbers: their order does not matter) and writes the stretch once.  A prompt's token sets a byte (all that do write the
// same), a generated one adds to its count.
__global__ void __launch_bounds__(RECORD_THREADS)
record_fresh_kernel(int* counts, uint32_t* seen, int n_slots, int V, int words, const int* slots, const int* starts,
                    const int* tokens, int n_tokens, const int* n_prompt, int cols) {
  mi_pdl_launch_dependents();
  extern __shared__ int4 record_smem[];
  int* tally = (int*)record_smem;                        // [cols]
  unsigned char* told = (unsigned char*)(tally + cols);  // [cols]
  const int req = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int begin = blockIdx.x * cols, n = min(V - begin, cols);
  for (int i = tid; i < cols * 5 / 16; i += RECORD_THREADS) record_smem[i] = make_int4(0, 0, 0, 0);
  mi_pdl_wait();
  const int slot = slots ? slots[req] : req;
  if (slot < 0 || slot >= n_slots) return;
  int first, last;
  long long made;
  tokens_of(req, starts, n_tokens, n_prompt, first, last, made);
  __syncthreads();
  for (int i0 = first + tid; i0 < last; i0 += 8 * RECORD_THREADS) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + u * RECORD_THREADS < last ? tokens[i0 + u * RECORD_THREADS] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const unsigned at = (unsigned)v[u] - (unsigned)begin;      // (a token below `begin` wraps to a large number)
      if (v[u] < 0 || at >= (unsigned)n) continue;
      if (i0 + u * RECORD_THREADS < made) told[at] = 1;
      else atomicAdd(&tally[at], 1);
    }
  }
  __syncthreads();
  int* c = counts + (size_t)slot * V + begin;
  uint32_t* s = seen + (size_t)slot * words + begin / 32;
  for (int i = tid; i < ((n + 31) & ~31); i += RECORD_THREADS) {
    const int k = tally[i];
    const unsigned bits = __ballot_sync(0xffffffffu, k > 0 || told[i]);
    if (i < n) c[i] = k;
    if (lane == 0) s[i >> 5] = bits;
  }
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
  if (V > 0x7fffffff - 65536 || n_tokens > 0x7fffffff - 65536) MI_REFUSE("record_tokens: vocabulary %d, %d tokens", V, n_tokens);
  const int words = (int)(((long long)V + 31) / 32);
  if (fresh) {
    // Every block of a request reads all its tokens: long stretches read them less often, short ones are more blocks.
    int cols = 16384;
    while (cols > 2048 && (long long)B * ((V + cols - 1) / cols) < 296) cols /= 2;
    static size_t allowed[64];
    const size_t smem = (size_t)cols * 5;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && smem > 48 * 1024 && dev >= 0 && dev < 64 && smem > allowed[dev]) {
      e = cudaFuncSetAttribute(record_fresh_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e == cudaSuccess) allowed[dev] = smem;
    }
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      MI_REFUSE("record_tokens: CUDA: %s", cudaGetErrorString(e));
    }
    MI_LAUNCH((record_fresh_kernel), dim3((V + cols - 1) / cols, B), RECORD_THREADS, smem, stream, counts, seen, n_slots, V,
              words, slots, starts, tokens, n_tokens, n_prompt, cols);
  } else {
    MI_LAUNCH((record_more_kernel), B, RECORD_THREADS, 0, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt);
  }
  MI_RETURN_LAUNCH_STATUS();
}
