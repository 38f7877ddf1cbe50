// Low-rank adapters of many requests beside a projection that all of them share:
//
//   out[t, c] = y[t, c] + sum_r (s_a (A_a x[t])[p(c), r]) B_a[c, r]        a = ids[t]
//   out[t, c] = y[t, c]                                                    where ids[t] is no adapter
//
// A projection may be several merged along its columns; column c belongs to part p(c), and every part has an A of its own:
// A is [adapters, parts, R, K], B [adapters, N, R].  Parts lie side by side, or (pairs) two of them alternate column by column.
// An adapter's own rank may be below R; what lies behind it is not read.  Sums are fp32.
#include "common.cuh"

MI_DEFINE_ERROR_API()

#define ADAPTER_MAX_PARTS 4
#define ADAPTER_THREADS 256

struct AdapterArgs {
  const void* x;
  long long ldx;
  const void* y;
  long long ldy;
  void* out;
  long long ldo;
  const void* a;
  const void* b;
  const int* ids;
  const int* ranks;
  const float* scale;
  float* h;                       // [M, P R]
  int M, N, K, n, P, R;
  int ends[ADAPTER_MAX_PARTS];    // where each part's columns end (side by side)
  int pairs;
  int chunks;                     // of columns (find_chunk)
  int vec;                        // 4 columns of y and out are one access
};

// One warp per (row, part and rank).
template <typename T>
__global__ void __launch_bounds__(ADAPTER_THREADS) adapter_shrink_kernel(const AdapterArgs g) {
  mi_pdl_enter();
  const int PR = g.P * g.R, lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * (ADAPTER_THREADS / 32) + (threadIdx.x >> 5);
  if (unit >= (long long)g.M * PR) return;
  const int t = (int)(unit / PR), pr = (int)(unit % PR);
  const int id = g.ids[t];
  if (id < 0 || id >= g.n) return;
  const int rank = g.ranks ? min(g.ranks[id], g.R) : g.R;
  if (pr % g.R >= rank) return;
  const T* x = (const T*)g.x + t * g.ldx;
  const T* a = (const T*)g.a + ((size_t)id * PR + pr) * g.K;
  float s = 0.f;
  for (int k = lane; k < g.K; k += 32) s = fmaf(mi_to_float(x[k]), mi_to_float(a[k]), s);
  s = mi_warp_sum(s);
  if (lane == 0) g.h[(size_t)t * PR + pr] = s * (g.scale ? g.scale[id] : 1.f);
}

template <typename T>
__global__ void __launch_bounds__(ADAPTER_THREADS) adapter_expand_kernel(const AdapterArgs g) {
  mi_pdl_enter();
  const int t = blockIdx.y, c = blockIdx.x * ADAPTER_THREADS + threadIdx.x;
  if (c >= g.N) return;
  const int id = g.ids[t];
  float s = mi_to_float(((const T*)g.y)[t * g.ldy + c]);
  if (id >= 0 && id < g.n) {
    const int rank = g.ranks ? min(g.ranks[id], g.R) : g.R;
    int p = 0;
    if (g.pairs) p = c & 1;
    else
      while (p + 1 < g.P && c >= g.ends[p]) ++p;
    const float* h = g.h + ((size_t)t * g.P + p) * g.R;
    const T* b = (const T*)g.b + ((size_t)id * g.N + c) * g.R;
    float d = 0.f;
    for (int r = 0; r < rank; ++r) d = fmaf(h[r], mi_to_float(b[r]), d);
    s += d;
  }
  ((T*)g.out)[t * g.ldo + c] = mi_from_float<T>(s);
}

// ---------------------------------------------------------------------------------------------- tensor cores, bfloat16
//
// Both products run on m16n8k16 with the adapter's rows (of A, then of B) as the 16 rows and tokens as the 8 columns, so that
// one token costs an eighth of a tile and not a sixteenth, and operands go from global memory to registers as they lie: a sum over
// k may take its terms in any order, so lane (g, t) = (lane / 4, lane % 4) loads 16 bytes, k = 8 t .. 8 t + 7, of row g, and
// its first two pairs are what the instruction wants for one step of 16 k, the other two for the next.

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 values of k: rows g (lo) and g + 8 (hi) of the one operand, token g of the other
__device__ __forceinline__ void mma_k32(float (&c)[4], const uint4& lo, const uint4& hi, const uint4& x) {
  mma_16816(c, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
  mma_16816(c, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
}

__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }
__device__ __forceinline__ uint4 load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

// The first `n` of eight bfloat16 values, zeros in the others' place (they may hold anything).
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
  if (n >= 8) return v;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (2 * i >= n) w[i] = 0u;
    else if (2 * i + 1 >= n) w[i] &= 0xffffu;
  }
  return v;
}

// A sum of the first product is held as two bfloat16 numbers, h = hi + lo, which leaves 2^-16 of it (as one, 2^-8): the second
// product runs twice, and the result is rounded once.
__device__ __forceinline__ void split_bf16(float v, bf16& hi, bf16& lo) {
  hi = __float2bfloat16_rn(v);
  // (an infinite value has no rest: inf - inf would make it NaN)
  const float rest = v - __bfloat162float(hi);
  lo = __float2bfloat16_rn(isinf(v) || isinf(__bfloat162float(hi)) ? 0.f : rest);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// a float of the same place in the shared memory of another block of the cluster
__device__ __forceinline__ float load_remote(const float* p, uint32_t rank) {
  uint32_t addr = (uint32_t)__cvta_generic_to_shared(p), there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

// The stride, in elements, of a token's row of h in shared memory: whole groups of 32 k, and 64 bytes off a multiple of 128,
// so that the 8 lanes of a quarter warp (2 tokens x 4 pieces of 16 bytes) touch all banks once.
__host__ __device__ inline int h_stride(int R) {
  const int r32 = (R + 31) / 32 * 32;
  return (r32 / 32) % 2 ? r32 : r32 + 32;
}

// Where a chunk of `size` columns lies: its part, first column and the part's end (pairs: one stretch of N columns).
__device__ __forceinline__ bool find_chunk(const AdapterArgs& g, int chunk, int size, int& part, int& c0, int& cend) {
  if (g.pairs) {
    part = 0;
    c0 = chunk * size;
    cend = g.N;
    return c0 < g.N;
  }
  int begin = 0;
  for (part = 0; part < g.P; ++part) {
    const int n = (g.ends[part] - begin + size - 1) / size;
    if (chunk < n) {
      c0 = begin + chunk * size;
      cend = g.ends[part];
      return true;
    }
    chunk -= n;
    begin = g.ends[part];
  }
  return false;
}
inline int count_chunks(const AdapterArgs& g, int size) {
  if (g.pairs) return (g.N + size - 1) / size;
  int n = 0, begin = 0;
  for (int p = 0; p < g.P; ++p) {
    n += (g.ends[p] - begin + size - 1) / size;
    begin = g.ends[p];
  }
  return n;
}

// ---- few rows: both products in one kernel, a cluster of blocks per adapter in use
//
// Every cluster takes up to 8 rows that share an adapter (or have none).  Its blocks cut K between them, exchange their shares of
// the first sums through distributed shared memory, and cut the columns of the result.  Nothing goes through global memory
// between the products and there is no second launch.

#define FEW_CLUSTER 8
#define FEW_THREADS 256
#define FEW_ROWS 8            // rows of a cluster
#define FEW_MAX 256           // rows of a call: one per thread in the search for a cluster's rows
#define FEW_GROUP 64          // sums of the first product that a pass makes
#define FEW_MAX_SUMS 1024     // parts * R

__global__ void __launch_bounds__(FEW_THREADS) adapter_few_kernel(const AdapterArgs g) {
  mi_pdl_enter();
  extern __shared__ __align__(16) unsigned char few_smem[];
  __shared__ uint32_t votes[FEW_THREADS / 32];
  __shared__ int rows[FEW_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int cand = blockIdx.x / FEW_CLUSTER, rank_in = (int)cluster_rank();
  const int PR = g.P * g.R, stride = h_stride(g.R);

  // The cluster stands for row `cand` and those behind it with the same adapter, if `cand` is the first, ninth, ... of them.
  int mine = tid < g.M ? g.ids[tid] : -1, id = g.ids[cand];
  if (mine < 0 || mine >= g.n) mine = -1;
  if (id < 0 || id >= g.n) id = -1;
  const bool match = tid < g.M && mine == id;
  const uint32_t vote = __ballot_sync(0xffffffffu, match);
  if (lane == 0) votes[warp] = vote;
  __syncthreads();
  int before = __popc(vote & ((1u << lane) - 1u)), at = 0;
  for (int w = 0; w < FEW_THREADS / 32; ++w) {
    if (w < warp) before += __popc(votes[w]);
    if (w < cand / 32) at += __popc(votes[w]);
    else if (w == cand / 32) at += __popc(votes[w] & ((1u << (cand & 31)) - 1u));
  }
  if (at % FEW_ROWS) return;                       // (all blocks of the cluster alike)
  int total = 0;
  for (int w = 0; w < FEW_THREADS / 32; ++w) total += __popc(votes[w]);
  const int count = min(FEW_ROWS, total - at);
  if (match && before >= at && before < at + FEW_ROWS) rows[before - at] = tid;
  __syncthreads();

  const bf16 *x = (const bf16*)g.x, *y = (const bf16*)g.y;
  bf16* out = (bf16*)g.out;
  int rank = id < 0 ? 0 : g.ranks ? max(0, min(g.ranks[id], g.R)) : g.R;
  if (rank == 0 && out == y) return;

  float* partial = (float*)few_smem;                                   // [warps][FEW_GROUP][FEW_ROWS]
  float* sums = partial + (FEW_THREADS / 32) * FEW_GROUP * FEW_ROWS;   // [PR][FEW_ROWS], this block's share of K
  bf16* h = (bf16*)(sums + PR * FEW_ROWS);                             // [P][hi, lo][FEW_ROWS][stride]

  if (rank > 0) {
    const int units = (g.K + 31) / 32;                                 // 32 values of k: 64 bytes of a row
    const int u0 = (int)((long long)units * rank_in / FEW_CLUSTER), u1 = (int)((long long)units * (rank_in + 1) / FEW_CLUSTER);
    const bf16* xr = x + (long long)rows[min(gq, count - 1)] * g.ldx + t * 8;
    const bf16* ad = (const bf16*)g.a + (size_t)id * PR * g.K + t * 8;
    for (int m0 = 0; m0 < PR; m0 += FEW_GROUP) {
      float acc[FEW_GROUP / 16][4];
#pragma unroll
      for (int m = 0; m < FEW_GROUP / 16; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
      bool have[FEW_GROUP / 16][2];
#pragma unroll
      for (int m = 0; m < FEW_GROUP / 16; ++m)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r = m0 + m * 16 + hf * 8 + gq;
          have[m][hf] = r < PR && r % g.R < rank;
        }
#pragma unroll 2
      for (int u = u0 + warp; u < u1; u += FEW_THREADS / 32) {
        const int k = u * 32 + t * 8;
        const bool in = k < g.K;
        const uint4 xv = in && gq < count ? load16(xr + u * 32) : zero4();
        uint4 av[FEW_GROUP / 16][2];
#pragma unroll
        for (int m = 0; m < FEW_GROUP / 16; ++m)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            av[m][hf] = in && have[m][hf] ? load16(ad + (size_t)(m0 + m * 16 + hf * 8 + gq) * g.K + u * 32) : zero4();
#pragma unroll
        for (int m = 0; m < FEW_GROUP / 16; ++m) mma_k32(acc[m], av[m][0], av[m][1], xv);
      }
      if (m0) __syncthreads();                     // the last pass's shares have been read
      float* mineP = partial + warp * FEW_GROUP * FEW_ROWS;
#pragma unroll
      for (int m = 0; m < FEW_GROUP / 16; ++m) {
        *reinterpret_cast<float2*>(mineP + (m * 16 + gq) * FEW_ROWS + 2 * t) = make_float2(acc[m][0], acc[m][1]);
        *reinterpret_cast<float2*>(mineP + (m * 16 + 8 + gq) * FEW_ROWS + 2 * t) = make_float2(acc[m][2], acc[m][3]);
      }
      __syncthreads();
      for (int i = tid; i < FEW_GROUP * FEW_ROWS && m0 * FEW_ROWS + i < PR * FEW_ROWS; i += FEW_THREADS) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_THREADS / 32; ++w) s += partial[w * FEW_GROUP * FEW_ROWS + i];
        sums[m0 * FEW_ROWS + i] = s;
      }
    }
    cluster_arrive();
    cluster_wait();
    const float scale = g.scale ? g.scale[id] : 1.f;
    for (int i = tid; i < g.P * FEW_ROWS * stride; i += FEW_THREADS) {
      const int p = i / (FEW_ROWS * stride), tok = i / stride % FEW_ROWS, r = i % stride;
      float s = 0.f;
      if (r < rank) {
#pragma unroll
        for (int c = 0; c < FEW_CLUSTER; ++c) s += load_remote(sums + (p * g.R + r) * FEW_ROWS + tok, c);
        s *= scale;
      }
      bf16 hi, lo;
      split_bf16(s, hi, lo);
      h[((p * 2 + 0) * FEW_ROWS + tok) * stride + r] = hi;
      h[((p * 2 + 1) * FEW_ROWS + tok) * stride + r] = lo;
    }
    cluster_arrive();                              // this block reads nobody's sums any more
    __syncthreads();
  }

  // 32 columns of up to 8 rows a warp and pass; lane (g, t) ends with columns 4 g .. 4 g + 3 of tokens 2 t and 2 t + 1.
  const int chunks = g.chunks;
  for (int chunk = rank_in * (FEW_THREADS / 32) + warp; chunk < chunks; chunk += FEW_CLUSTER * (FEW_THREADS / 32)) {
    int part, c0, cend;
    if (!find_chunk(g, chunk, 32, part, c0, cend)) break;
    const int c = c0 + 4 * gq;
    float acc[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
    const bf16* b = (const bf16*)g.b + ((size_t)max(id, 0) * g.N + c) * g.R + t * 8;
    for (int k0 = 0; k0 < rank; k0 += 32) {
      const int n = rank - k0 - t * 8;             // values of this lane's piece that there are
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint4 w[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int j = 2 * hf + m;                // column 4 g + j
          w[hf] = n > 0 && c + j < cend ? first_of(load16(b + (size_t)j * g.R + k0), n) : zero4();
        }
        const bf16* hp = h + ((g.pairs ? m : part) * 2 * FEW_ROWS + gq) * stride + k0 + t * 8;
        mma_k32(acc[m], w[0], w[1], load16(hp));
        mma_k32(acc[m], w[0], w[1], load16(hp + FEW_ROWS * stride));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tok = 2 * t + i;
      if (tok >= count) continue;
      const long long row = rows[tok];
      const bf16* yp = y + row * g.ldy + c;
      bf16* op = out + row * g.ldo + c;
      const float d[4] = {acc[0][i], acc[1][i], acc[0][2 + i], acc[1][2 + i]};
      if (g.vec && c + 4 <= cend) {
        Vec4<bf16> v;
        float f[4];
        v.load(yp);
        if (rank > 0) {
          v.get(f);
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] += d[j];
          v.set(f);
        }
        v.store(op);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < cend) op[j] = rank > 0 ? __float2bfloat16_rn(__bfloat162float(yp[j]) + d[j]) : yp[j];
      }
    }
  }
  __syncwarp();
  if (rank > 0) cluster_wait();                    // the block's shared memory stays until all have read it
}

static size_t few_smem_bytes(int P, int R) {
  return (size_t)(FEW_THREADS / 32) * FEW_GROUP * FEW_ROWS * 4 + (size_t)P * R * FEW_ROWS * 4 +
         (size_t)P * 2 * FEW_ROWS * h_stride(R) * 2;
}

static int refused_by_cuda(cudaError_t e) {
  (void)cudaGetLastError();
  snprintf(g_mi_error, sizeof(g_mi_error), "CUDA: %s", cudaGetErrorString(e));
  return (int)e;
}

template <typename K>
static cudaError_t launch_cluster(K kernel, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                                  const AdapterArgs& g) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = mi_pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, g);
}
// Dynamic shared memory over 48 KB is allowed once per kernel and device.
template <typename K>
static cudaError_t allow_smem(K kernel, size_t bytes, size_t* allowed) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || bytes <= 48 * 1024 || bytes <= allowed[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) allowed[dev] = bytes;
  return e;
}

extern "C" int mi_adapter_add(const void* y, long long ldy, const void* x, long long ldx, const void* a, const void* b,
                              void* out, long long ldo, const int* ids, const float* scale, const int* ranks, float* h, int M,
                              int N, int K, int n, int P, int R, int end0, int end1, int end2, int end3, int pairs, int dtype,
                              cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (M > 65535) MI_REFUSE("adapter_add: %d rows, at most 65535", M);
  if (P < 1 || P > ADAPTER_MAX_PARTS) MI_REFUSE("adapter_add: %d parts, at most %d", P, ADAPTER_MAX_PARTS);
  AdapterArgs g = {x, ldx, y, ldy, out, ldo, a, b, ids, ranks, scale, h, M, N, K, n, P, R, {end0, end1, end2, end3}, pairs, 0, 0};
  // The tensor-core kernels take rows of x, A and B in pieces of 16 bytes.
  const bool pieces = dtype == MI_DTYPE_BF16 && n > 0 && R > 0 && K > 0 && R % 8 == 0 && K % 8 == 0 && mi_aligned(a, 16) &&
                      mi_aligned(b, 16) && mi_aligned(x, 16) && (M == 1 || ldx % 8 == 0);
  bool starts4 = true;
  for (int p = 0; p + 1 < P && !pairs; ++p) starts4 = starts4 && g.ends[p] % 4 == 0;
  g.vec = starts4 && mi_aligned(y, 8) && mi_aligned(out, 8) && (M == 1 || (ldy % 4 == 0 && ldo % 4 == 0));
  if (pieces && M <= FEW_MAX && P * R <= FEW_MAX_SUMS) {
    static size_t allowed[64];
    const size_t smem = few_smem_bytes(P, R);
    g.chunks = count_chunks(g, 32);
    cudaError_t e = allow_smem(adapter_few_kernel, smem, allowed);
    if (e == cudaSuccess) e = launch_cluster(adapter_few_kernel, dim3(M * FEW_CLUSTER), FEW_THREADS, smem, FEW_CLUSTER, stream, g);
    if (e != cudaSuccess) return refused_by_cuda(e);
    MI_RETURN_LAUNCH_STATUS();
  }
  const long long units = (long long)M * P * R, per = ADAPTER_THREADS / 32;
  if ((units + per - 1) / per > 0x7fffffffLL) MI_REFUSE("adapter_add: %lld sums of the first product", units);
  const unsigned blocks = n > 0 ? (unsigned)((units + per - 1) / per) : 0u;
  const dim3 grid((N + ADAPTER_THREADS - 1) / ADAPTER_THREADS, M);
  if (dtype == MI_DTYPE_F32) {
    if (blocks) MI_LAUNCH((adapter_shrink_kernel<float>), blocks, ADAPTER_THREADS, 0, stream, g);
    MI_LAUNCH((adapter_expand_kernel<float>), grid, ADAPTER_THREADS, 0, stream, g);
  } else {
    if (blocks) MI_LAUNCH((adapter_shrink_kernel<bf16>), blocks, ADAPTER_THREADS, 0, stream, g);
    MI_LAUNCH((adapter_expand_kernel<bf16>), grid, ADAPTER_THREADS, 0, stream, g);
  }
  MI_RETURN_LAUNCH_STATUS();
}
