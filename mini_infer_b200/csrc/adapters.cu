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

extern "C" int mi_adapter_add(const void* y, long long ldy, const void* x, long long ldx, const void* a, const void* b,
                              void* out, long long ldo, const int* ids, const float* scale, const int* ranks, float* h, int M,
                              int N, int K, int n, int P, int R, int end0, int end1, int end2, int end3, int pairs, int dtype,
                              cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (M > 65535) MI_REFUSE("adapter_add: %d rows, at most 65535", M);
  if (P < 1 || P > ADAPTER_MAX_PARTS) MI_REFUSE("adapter_add: %d parts, at most %d", P, ADAPTER_MAX_PARTS);
  AdapterArgs g = {x, ldx, y, ldy, out, ldo, a, b, ids, ranks, scale, h, M, N, K, n, P, R, {end0, end1, end2, end3}, pairs};
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
