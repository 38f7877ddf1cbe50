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

#define ADJUST_THREADS 128
#define ADJUST_GROUPS 8                         // groups of 4 columns of a lane: a word of bits per lane, in other order
#define ADJUST_WARP_COLS (32 * ADJUST_GROUPS * 4)

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

// Bound by memory: a logit is read and written once, and each seen bit, mask bit, bias and the count of a seen token read once; the
// operations are a few a column.  A warp takes 1024 columns of a row.  All of them pass through in groups of four a lane, eight loads
// under way at once, with minus infinity put in by the mask's bits; what else changes are single columns, and they are done on their
// own behind that: each lane goes through the seen bits of one word (32 columns; where one has many, they are shared out among the
// lanes), four at a time, and the warp through the row's biases.  So the way of the many columns that stay as they are is a load, a few
// bits and a store.  A row that starts off a 16-byte boundary is taken from its first boundary on; the up to three columns in front
// are the first warp's.  In place, columns that do not change are neither read nor written.
//
// 256 rows of 128256 with histories of up to 1000 tokens and 100 biases each, out of place: 49 us, 5.4 TB/s (a thread per column
// with its bits and count 130 us); 16 rows with histories of up to 1500 5.7 us; one row of 32000 with everything 3.5 us, which is
// launch and latency.  Blocks of four warps: of eight, whose rows and tails share out worse, 53, 6.4 and 3.7 us.
template <bool IN_PLACE>
__global__ void __launch_bounds__(ADJUST_THREADS) adjust_logits_kernel(const AdjustArgs a) {
  mi_pdl_enter();   // the logits and the histories come from the kernels before this one
  __shared__ unsigned short lists[ADJUST_THREADS / 32][ADJUST_WARP_COLS];
  const int row = blockIdx.y, lane = threadIdx.x & 31;
  const int part = blockIdx.x * (ADJUST_THREADS / 32) + (threadIdx.x >> 5);
  const float* in = a.logits + (size_t)row * a.ld_in;
  float* out = a.out + (size_t)row * a.ld_out;
  const bool biases = a.bias_starts != nullptr;
  const int slot = a.seen ? (a.slots ? a.slots[row] : row) : -1;
  const int mrow = a.masks ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
  const int first = biases ? max(0, a.bias_starts[row]) : 0, last = biases ? min(a.n_bias, a.bias_starts[row + 1]) : 0;
  // the columns before the first 16-byte boundary; this warp's: [start, end)
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / 4;
  const int start = part * ADJUST_WARP_COLS + head, end = min(a.V, start + ADJUST_WARP_COLS);
  const int lead = part ? 0 : min(head, a.V);
  if (start >= end && !lead) return;

  float4 z[ADJUST_GROUPS];
  if (!IN_PLACE) {
#pragma unroll
    for (int j = 0; j < ADJUST_GROUPS; ++j) {
      const int c = start + j * 128 + lane * 4;
      if (c + 4 <= end) z[j] = *reinterpret_cast<const float4*>(in + c);
    }
  }
  const bool known = slot >= 0 && slot < a.n_slots, masked = mrow >= 0 && mrow < a.n_masks;
  const uint32_t* seen = a.seen + (size_t)(known ? slot : 0) * a.words;
  const uint32_t* mask = a.masks + (size_t)(masked ? mrow : 0) * a.words;
  const int* counts = known && a.counts ? a.counts + (size_t)slot * a.V : nullptr;
  const float rep = known && a.repetition ? a.repetition[row] : 1.f;
  const float pres = known && a.presence ? a.presence[row] : 0.f;
  const float freq = known && a.frequency ? a.frequency[row] : 0.f;
  int ids[4];
  float values[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int j = first + 32 * u + lane;
    ids[u] = j < last ? a.bias_ids[j] : -1;
    values[u] = j < last ? a.bias_values[j] : 0.f;
  }

  // the lane's word: columns mine .. mine + 31
  const int mine = start + lane * 32, w = mine >> 5;
  uint32_t told = 0u, shut = 0u;
  if (mine < end) {
    const uint32_t valid = end - mine >= 32 ? ~0u : (1u << (end - mine)) - 1u;
    const int w1 = head ? min(w + 1, a.words - 1) : w;
    if (known) told = __funnelshift_r(seen[w], seen[w1], head) & valid;
    if (masked) shut = ~__funnelshift_r(mask[w], mask[w1], head) & valid;
  }
  const bool any_shut = __any_sync(0xffffffffu, shut != 0u);
  if (!IN_PLACE || any_shut) {
    const bool vec_out = (reinterpret_cast<uintptr_t>(out + start) & 15) == 0;
#pragma unroll
    for (int j = 0; j < ADJUST_GROUPS; ++j) {
      const int c = start + j * 128 + lane * 4;
      const uint32_t four = any_shut ? (__shfl_sync(0xffffffffu, shut, j * 4 + (lane >> 3)) >> ((lane & 7) * 4)) & 15u : 0u;
      if (IN_PLACE ? four == 15u && vec_out : c + 4 <= end && vec_out) {
        float4 v = IN_PLACE ? make_float4(0.f, 0.f, 0.f, 0.f) : z[j];
        if (four & 1u) v.x = -INFINITY;
        if (four & 2u) v.y = -INFINITY;
        if (four & 4u) v.z = -INFINITY;
        if (four & 8u) v.w = -INFINITY;
        *reinterpret_cast<float4*>(out + c) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (IN_PLACE ? (four >> i) & 1u : c + i < end) out[c + i] = (four >> i) & 1u ? -INFINITY : in[c + i];
      }
    }
  }
  const auto penalised = [&](float v, int n) {
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    if (n > 0) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)n)), pres);
    return v;
  };
  if (lane < lead) {
    const bool closed = masked && !((mask[0] >> lane) & 1u), here = known && ((seen[0] >> lane) & 1u);
    if (closed) out[lane] = -INFINITY;
    else if (here) out[lane] = penalised(in[lane], counts ? counts[lane] : 0);
    else if (!IN_PLACE) out[lane] = in[lane];
  }
  __syncwarp();
  // Where a word has many, the columns of all lanes are listed in shared memory first and shared out evenly.
  uint32_t left = told & ~shut;
  int todo = __popc(left), listed = 0;
  if (__any_sync(0xffffffffu, todo > 4)) {
    unsigned short* list = lists[threadIdx.x >> 5];
    int at = todo;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += n;
    }
    listed = __shfl_sync(0xffffffffu, at, 31);
    for (at -= todo; left; left &= left - 1u) list[at++] = (unsigned short)(lane * 32 + __ffs(left) - 1);
    __syncwarp();
    for (int j = lane; j < listed; j += 128) {
      int c[4], n[4];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = j + 32 * i < listed ? start + list[j + 32 * i] : -1;
        v[i] = c[i] >= 0 ? in[c[i]] : 0.f;
        n[i] = c[i] >= 0 && counts ? counts[c[i]] : 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c[i] >= 0) out[c[i]] = penalised(v[i], n[i]);
    }
  } else if (left) {
    int c[4], n[4];
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = left ? mine + __ffs(left) - 1 : -1;
      left &= left - 1u;
      v[i] = c[i] >= 0 ? in[c[i]] : 0.f;
      n[i] = c[i] >= 0 && counts ? counts[c[i]] : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c[i] >= 0) out[c[i]] = penalised(v[i], n[i]);
  }
  // The biases in the order of the list: of equal ids within 32 entries the first one's lane adds all, so that every sum has
  // one order.
  const int from = part ? start : 0;
  for (int j0 = first; j0 < last; j0 += 128) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int v = ids[u];
      const bool ours = v >= from && v < end && (!masked || ((mask[v >> 5] >> (v & 31)) & 1u));
      unsigned any = __ballot_sync(0xffffffffu, ours);
      if (any) {
        __syncwarp();                             // what other lanes have written of these columns
        const unsigned same = __match_any_sync(0xffffffffu, ours ? v : -1 - lane);
        const bool leads = ours && lane == __ffs(same) - 1;
        float sum = leads ? out[v] : 0.f;
        while (any) {
          const int l = __ffs(any) - 1;
          any &= any - 1;
          const float add = __shfl_sync(0xffffffffu, values[u], l);
          if (leads && ((same >> l) & 1u)) sum = __fadd_rn(sum, add);
        }
        if (leads) out[v] = sum;
        __syncwarp();
      }
      const int j = j0 + 128 + 32 * u + lane;
      ids[u] = j < last ? a.bias_ids[j] : -1;
      values[u] = j < last ? a.bias_values[j] : 0.f;
    }
  }
}

// The arguments of a call as one block of 64-bit numbers.
struct AdjustCall {
  long long logits, ld_in, out, ld_out, B, V, slots, seen, counts, n_slots, repetition, presence, frequency, bias_starts, bias_ids,
      bias_values, n_bias, masks, mask_rows, n_masks;
};

extern "C" int mi_adjust_logits(const AdjustCall* call, cudaStream_t stream) {
  const AdjustCall& c = *call;
  const long long B = c.B, V = c.V, n_bias = c.n_bias;
  if (B <= 0 || V <= 0) return 0;
  if (n_bias > 0x7fffffff - 65536) MI_REFUSE("adjust_logits: %lld biases", n_bias);
  if (B > 65535) MI_REFUSE("adjust_logits: %lld rows, at most 65535", B);
  if (V > 0x7fffffff - 65536) MI_REFUSE("adjust_logits: vocabulary %lld", V);
  const bool in_place = c.out == c.logits;
  const AdjustArgs a = {(const float*)c.logits, (float*)c.out, c.ld_in, c.ld_out, (int)V, (int)((V + 31) / 32), (const int*)c.slots,
                        (const uint32_t*)c.seen, (const int*)c.counts, (int)c.n_slots, (const float*)c.repetition,
                        (const float*)c.presence, (const float*)c.frequency, (const int*)c.bias_starts, (const int*)c.bias_ids,
                        (const float*)c.bias_values, (int)n_bias, (const uint32_t*)c.masks, (const int*)c.mask_rows, (int)c.n_masks};
  const int cols = ADJUST_WARP_COLS * (ADJUST_THREADS / 32);
  const dim3 grid((unsigned)((V + cols - 1) / cols), (unsigned)B);
  if (in_place)
    MI_LAUNCH((adjust_logits_kernel<true>), grid, ADJUST_THREADS, 0, stream, a);
  else
    MI_LAUNCH((adjust_logits_kernel<false>), grid, ADJUST_THREADS, 0, stream, a);
  MI_RETURN_LAUNCH_STATUS();
}

// ---------------------------------------------------------------------------------------------- histories

#define RECORD_THREADS 256      // of a block that adds tokens
#define RECORD_AHEAD 4

// Tokens [first, last) are the request's (without `starts`: one token each), those from `made` on are generated ones.
__device__ __forceinline__ void tokens_of(int req, const int* starts, int n_tokens, const int* n_prompt, int& first, int& last,
                                          long long& made) {
  const int from = starts ? starts[req] : req;
  first = max(0, from);
  last = min(n_tokens, starts ? starts[req + 1] : req + 1);
  made = n_prompt ? (long long)from + n_prompt[req] : from;
}

// op(token) for the tokens [lo, hi), four to a load where they lie on a 16-byte boundary, several loads under way at once.
template <int THREADS, typename F>
__device__ __forceinline__ void scan_tokens(const int* tokens, int lo, int hi, int tid, F op) {
  if (lo >= hi) return;
  const int to_boundary = (int)((16 - (reinterpret_cast<uintptr_t>(tokens + lo) & 15)) & 15) / 4;
  const int a = min(hi, lo + to_boundary), n4 = (hi - a) >> 2;
  if (tid < a - lo) op(tokens[lo + tid]);
  const int4* p = reinterpret_cast<const int4*>(tokens + a);
  for (int j0 = tid; j0 < n4; j0 += RECORD_AHEAD * THREADS) {
    int4 v[RECORD_AHEAD];
#pragma unroll
    for (int u = 0; u < RECORD_AHEAD; ++u) v[u] = j0 + u * THREADS < n4 ? p[j0 + u * THREADS] : make_int4(-1, -1, -1, -1);
#pragma unroll
    for (int u = 0; u < RECORD_AHEAD; ++u) {
      op(v[u].x);
      op(v[u].y);
      op(v[u].z);
      op(v[u].w);
    }
  }
  if (tid < hi - a - 4 * n4) op(tokens[a + 4 * n4 + tid]);
}

// A history written anew, bound by the bytes that it has, 4 1/8 a token of the vocabulary, and where prompts are long by the tokens that
// every block of a request reads again (from L2): the block counts the request's tokens within its stretch of the vocabulary in shared memory
// (whole numbers: their order does not matter) and writes the stretch once.  A prompt's token sets a byte (all that do write the
// same), a generated one adds to its count.
template <int THREADS>
__global__ void __launch_bounds__(THREADS)
record_fresh_kernel(int* counts, uint32_t* seen, int n_slots, int V, int words, const int* slots, const int* starts,
                    const int* tokens, int n_tokens, const int* n_prompt, int cols) {
  mi_pdl_launch_dependents();
  extern __shared__ int4 record_smem[];
  int* tally = (int*)record_smem;                        // [cols]
  unsigned char* told = (unsigned char*)(tally + cols);  // [cols]
  const int req = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int begin = blockIdx.x * cols, n = min(V - begin, cols);
  for (int i = tid; i < cols * 5 / 16; i += THREADS) record_smem[i] = make_int4(0, 0, 0, 0);
  mi_pdl_wait();
  const int slot = slots ? slots[req] : req;
  if (slot < 0 || slot >= n_slots) return;
  int first, last;
  long long made;
  tokens_of(req, starts, n_tokens, n_prompt, first, last, made);
  const int turn = (int)max((long long)first, min(made, (long long)last));
  __syncthreads();
  // (a token below `begin` wraps to a large number, and so does a negative one, but for a block that begins above 2^31)
  scan_tokens<THREADS>(tokens, first, turn, tid, [&](int v) {
    const unsigned at = (unsigned)v - (unsigned)begin;
    if (at < (unsigned)n) told[at] = 1;
  });
  scan_tokens<THREADS>(tokens, turn, last, tid, [&](int v) {
    const unsigned at = (unsigned)v - (unsigned)begin;
    if (at < (unsigned)n) atomicAdd(&tally[at], 1);
  });
  __syncthreads();
  int* c = counts + (size_t)slot * V + begin;
  uint32_t* s = seen + (size_t)slot * words + begin / 32;
  for (int i = tid; i < ((n + 31) & ~31); i += THREADS) {
    const int k = tally[i];
    const unsigned bits = __ballot_sync(0xffffffffu, k > 0 || told[i]);
    if (i < n) c[i] = k;
    if (lane == 0) s[i >> 5] = bits;
  }
}

// Tokens added to what a history holds, RECORD_EACH a thread; a step's one token for each of 64 requests is a launch and three
// dependent loads, 1.5 us.  A frequent token's bit is mostly there already: it is looked at
// (in L2, where the others set it) before it is set.
#define RECORD_EACH 4
__global__ void __launch_bounds__(RECORD_THREADS)
record_more_kernel(int* counts, uint32_t* seen, int n_slots, int V, int words, const int* slots, const int* starts,
                   const int* tokens, int n_tokens, const int* n_prompt, int B) {
  mi_pdl_enter();
  const int i0 = blockIdx.x * (RECORD_THREADS * RECORD_EACH) + threadIdx.x;
  int v[RECORD_EACH];
#pragma unroll
  for (int u = 0; u < RECORD_EACH; ++u) v[u] = i0 + u * RECORD_THREADS < n_tokens ? tokens[i0 + u * RECORD_THREADS] : -1;
  const int begins = starts ? starts[0] : 0;
#pragma unroll
  for (int u = 0; u < RECORD_EACH; ++u) {
    const int i = i0 + u * RECORD_THREADS;
    if (v[u] < 0 || v[u] >= V || i < begins) continue;
    int req = i;                                         // the last request that begins at or before token i
    if (starts) {
      int hi = B;
      for (req = 0; hi - req > 1;) {
        const int mid = (req + hi) >> 1;
        if (starts[mid] <= i) req = mid;
        else hi = mid;
      }
      if (i >= starts[req + 1]) continue;
    }
    if (req >= B) continue;
    const int slot = slots ? slots[req] : req;
    if (slot < 0 || slot >= n_slots) continue;
    uint32_t* word = seen + (size_t)slot * words + (v[u] >> 5);
    const uint32_t bit = 1u << (v[u] & 31);
    if (!(__ldcg(word) & bit)) atomicOr(word, bit);
    if (!n_prompt || i >= (long long)(starts ? starts[req] : i) + n_prompt[req]) atomicAdd(&counts[(size_t)slot * V + v[u]], 1);
  }
}

struct RecordCall {
  long long counts, seen, n_slots, V, slots, starts, tokens, n_tokens, n_prompt, B, fresh;
};

extern "C" int mi_record_tokens(const RecordCall* call, cudaStream_t stream) {
  const RecordCall& c = *call;
  if (c.B > 65535) MI_REFUSE("record_tokens: %lld requests, at most 65535", c.B);
  if (c.V > 0x7fffffff - 65536 || c.n_tokens > 0x7fffffff - 65536 || c.n_slots > 0x7fffffff)
    MI_REFUSE("record_tokens: vocabulary %lld, %lld tokens, %lld histories", c.V, c.n_tokens, c.n_slots);
  int* counts = (int*)c.counts;
  uint32_t* seen = (uint32_t*)c.seen;
  const int *slots = (const int*)c.slots, *starts = (const int*)c.starts, *tokens = (const int*)c.tokens, *n_prompt = (const int*)c.n_prompt;
  const int n_slots = (int)c.n_slots, V = (int)c.V, n_tokens = (int)c.n_tokens, B = (int)c.B, fresh = c.fresh != 0;
  if (B <= 0 || V <= 0) return 0;
  const int words = (int)(((long long)V + 31) / 32);
  if (!fresh) {
    const int blocks = (n_tokens + RECORD_THREADS * RECORD_EACH - 1) / (RECORD_THREADS * RECORD_EACH);
    if (!blocks) return 0;
    MI_LAUNCH((record_more_kernel), blocks, RECORD_THREADS, 0, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt, B);
    MI_RETURN_LAUNCH_STATUS();
  }
  // Every block of a request reads all its tokens: long stretches read them less often, short ones are more blocks.  64 requests
  // of 128256 tokens each, us with stretches of 16384 (1024 threads), 8192 (512) and 4096 (512): up to 32768 tokens 17.6, 19.2
  // and 26.8; 100 tokens 12.6, 11.4 and 14.8; 16 requests of up to 2048 tokens 5.6, 4.9 and 4.6; one of 17 and a vocabulary of 32000
  // 3.6, 2.9 and 2.4, and 2.2 with 2048 (256).
  const bool many = n_tokens / B > 8192;
  int cols = many ? 16384 : 8192;
  while (cols > 2048 && (long long)B * ((V + cols - 1) / cols) < 2 * 148) cols /= 2;
  const int threads = many ? 1024 : cols >= 4096 ? 512 : 256;
  const size_t smem = (size_t)cols * 5;
  const dim3 grid((V + cols - 1) / cols, B);
  if (threads == 1024) {
    static bool allowed[64];                  // more than 48 KB, once per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(dev < 64 && allowed[dev])) {
      e = cudaFuncSetAttribute(record_fresh_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 5);
      if (e == cudaSuccess && dev < 64) allowed[dev] = true;
    }
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      MI_REFUSE("record_tokens: CUDA: %s", cudaGetErrorString(e));
    }
    MI_LAUNCH((record_fresh_kernel<1024>), grid, threads, smem, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt, cols);
  } else if (threads == 512) {
    MI_LAUNCH((record_fresh_kernel<512>), grid, threads, smem, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt, cols);
  } else {
    MI_LAUNCH((record_fresh_kernel<256>), grid, threads, smem, stream, counts, seen, n_slots, V, words, slots, starts, tokens,
              n_tokens, n_prompt, cols);
  }
  MI_RETURN_LAUNCH_STATUS();
}
