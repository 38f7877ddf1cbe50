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
  int vec;                        // 4 columns of y and out are one access
  int span;                       // columns of a block
  int ks;                         // parts of the sum over K
  const int* order;
  const int4* items;
  int constant;                   // no kernel in flight writes A and B
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

// ---- items: up to 8 NT rows that share an adapter (or have none)
//
// For up to FEW_MAX rows every block finds its item in the ids; for more, adapter_plan has put the rows in order.

#define TILE_THREADS 256
#define TILE_WARPS (TILE_THREADS / 32)
#define FEW_MAX 128           // rows of a call whose items the blocks find by themselves
#define SUM_GROUP 64          // sums of the first product that a block makes
#define MAX_ROWS 64           // of an item

struct Item {
  int id, count;              // adapter (-1: none), rows
};

// Item `index` of a call of few rows, 8 rows each: rows with one adapter are put together in their order, and items are in the order of
// their first rows.  `rows` and `ids` are shared memory; count 0: there is no such item.
__device__ __forceinline__ Item few_item(const AdapterArgs& g, int index, int* rows, int* ids, int* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int id = -1;
  if (tid < FEW_MAX) {
    id = tid < g.M ? __ldcg(g.ids + tid) : -2;
    if (id >= g.n || id < -1) id = tid < g.M ? -1 : -2;
    ids[tid] = id;
  }
  if (tid < 2) found[tid] = 0;
  __syncthreads();
  int before = 0;                                   // earlier rows with this adapter
  if (tid < g.M) {
    const int4* p = reinterpret_cast<const int4*>(ids);
    for (int j = 0; j < tid / 4; ++j) {
      const int4 v = p[j];
      before += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
    }
    for (int j = tid & ~3; j < tid; ++j) before += ids[j] == id;
  }
  const bool leads = tid < g.M && before % 8 == 0;
  const unsigned vote = __ballot_sync(0xffffffffu, leads);
  int* votes = ids + FEW_MAX;                       // [warps]
  if (lane == 0) votes[warp] = __popc(vote);
  __syncthreads();
  int at = __popc(vote & ((1u << lane) - 1u));
  for (int w = 0; w < warp; ++w) at += votes[w];
  if (leads && at == index) {
    found[0] = id + 2;
    found[1] = before;
  }
  __syncthreads();
  Item item = {found[0] - 2, 0};
  const int base = found[1];
  const bool mine = tid < g.M && found[0] && id == item.id && before >= base && before < base + 8;
  if (mine) rows[before - base] = tid;
  item.count = __syncthreads_count(mine);
  return item;
}

template <int NT>
__device__ __forceinline__ Item get_item(const AdapterArgs& g, int index, int* rows, int* ids, int* found) {
  if (NT == 1) return few_item(g, index, rows, ids, found);
  const int4 v = __ldcg(g.items + index);
  if (threadIdx.x < (unsigned)v.z) rows[threadIdx.x] = __ldcg(g.order + v.y + threadIdx.x);
  __syncthreads();
  return Item{v.x, v.z};
}

__device__ __forceinline__ int rank_of(const AdapterArgs& g, int id) {
  return id < 0 ? 0 : g.ranks ? max(0, min(__ldcg(g.ranks + id), g.R)) : g.R;
}

// ---- the first product: a block makes SUM_GROUP sums of an item over a share of K.  NT: 8-token columns of tiles of an item.
//
// Warps cut the share of K between them (with 64 tokens, four ways, and the tokens two ways), their sums meet in shared memory
// and go to h as one part of the sum over K.

template <int NT>
__global__ void __launch_bounds__(TILE_THREADS, NT == 1 ? 2 : 1) adapter_sums_kernel(const AdapterArgs g) {
  constexpr int TW = NT == 1 ? 1 : 2, KW = TILE_WARPS / TW, NW = NT / TW, TOK = 8 * NT, MT = SUM_GROUP / 16, PAD = SUM_GROUP + 4;
  // The kernel behind this one starts once the ids and operands of both are there; it waits for these sums alone.
  mi_pdl_wait();
  mi_pdl_launch_dependents();
  extern __shared__ __align__(16) float sums_smem[];          // [KW][TOK][PAD]
  __shared__ int rows[MAX_ROWS];
  __shared__ __align__(16) int ids[FEW_MAX + TILE_WARPS];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int kw = warp % KW, tw = warp / KW;
  const Item item = get_item<NT>(g, blockIdx.y, rows, ids, found);
  const int rank = rank_of(g, item.id);
  if (item.count == 0 || rank == 0) return;
  const int PR = g.P * g.R, m0 = blockIdx.z * SUM_GROUP;
  const int units = (g.K + 31) / 32;                          // 32 values of k: 64 bytes of a row
  const int u0 = (int)((long long)units * blockIdx.x / g.ks), u1 = (int)((long long)units * (blockIdx.x + 1) / g.ks);

  const bf16* xr[NW];
  bool live[NW];
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    const int tok = (tw * NW + j) * 8 + gq;
    live[j] = tok < item.count;
    xr[j] = (const bf16*)g.x + (long long)rows[live[j] ? tok : 0] * g.ldx + t * 8;
  }
  const bf16* ar = (const bf16*)g.a + ((size_t)item.id * PR + m0 + gq) * g.K + t * 8;
  bool have[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = m0 + m * 16 + hf * 8 + gq;
      have[m][hf] = r < PR && r % g.R < rank;
    }
  float acc[MT][NW][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
  // The operands of the next 32 k are loaded before the products of the last ones.
  uint4 xv[NW], av[MT][2];
  const auto load = [&](int u, uint4 (&xn)[NW], uint4 (&an)[MT][2]) {
    const bool in = u < u1 && u * 32 + t * 8 < g.K;
#pragma unroll
    for (int j = 0; j < NW; ++j) xn[j] = in && live[j] ? load16(xr[j] + u * 32) : zero4();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        an[m][hf] = in && have[m][hf] ? load16(ar + (size_t)(m * 16 + hf * 8) * g.K + u * 32) : zero4();
  };
  load(u0 + kw, xv, av);
  for (int u = u0 + kw; u < u1; u += KW) {
    uint4 xn[NW], an[MT][2];
    load(u + KW, xn, an);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NW; ++j) mma_k32(acc[m][j], av[m][0], av[m][1], xv[j]);
#pragma unroll
    for (int j = 0; j < NW; ++j) xv[j] = xn[j];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      av[m][0] = an[m][0];
      av[m][1] = an[m][1];
    }
  }
  float* mine = sums_smem + (kw * TOK + tw * NW * 8) * PAD;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(j * 8 + 2 * t + (i & 1)) * PAD + m * 16 + (i >> 1) * 8 + gq] = acc[m][j][i];
  __syncthreads();
  float* h = g.h + (size_t)blockIdx.x * g.M * PR + m0;
  for (int i = tid; i < item.count * (SUM_GROUP / 4); i += TILE_THREADS) {
    const int tok = i / (SUM_GROUP / 4), r = i % (SUM_GROUP / 4) * 4;
    if (m0 + r >= PR) continue;                               // (PR is a multiple of 8)
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(sums_smem + (w * TOK + tok) * PAD + r);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<float4*>(h + (size_t)rows[tok] * PR + r) = s;
  }
}

// ---- the second product and the sum with y: a warp takes 32 columns of 8 or 32 rows at a time; lane (g, t) ends with columns
// 4 g .. 4 g + 3 of tokens 2 t and 2 t + 1 of every 8.  B and y of the next columns are loaded between the products and the
// stores of the last ones.
//
// KG: groups of 32 k (0: as many as there are).  FOLD (up to 16 k): the rests of the sums stand where the second 16 k of a group would, so
// that one pass does for both.

template <int NT, int KG, bool FOLD>
__global__ void __launch_bounds__(TILE_THREADS, NT == 1 ? 3 : 2) adapter_add_kernel(const AdapterArgs g) {
  constexpr int TW = NT == 1 ? 1 : 2, CW = TILE_WARPS / TW, NW = NT / TW, TOK = 8 * NT;
  extern __shared__ __align__(16) unsigned char add_smem[];
  bf16* h = (bf16*)add_smem;                                  // [parts of the block][hi, lo][TOK][stride]
  __shared__ int rows[MAX_ROWS];
  __shared__ long long y_at[TOK], out_at[TOK];                // where the rows begin
  __shared__ __align__(16) int ids[FEW_MAX + TILE_WARPS];
  __shared__ int found[2];
  mi_pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int cw = warp % CW, tok0 = warp / CW * NW * 8;
  // (the kernel in front was started behind everything that wrote the ids and the operands, and started this one behind that)
  const Item item = get_item<NT>(g, blockIdx.y, rows, ids, found);
  const int rank = rank_of(g, item.id), R = g.R;
  const bf16* y = (const bf16*)g.y;
  bf16* out = (bf16*)g.out;
  int part, c_first, c_end;
  const bool there = find_chunk(g, blockIdx.x, g.span, part, c_first, c_end) && item.count > 0 && (rank > 0 || out != y);
  c_end = min(c_end, c_first + g.span);
  const int PR = g.P * R, stride = h_stride(R), np = g.pairs ? 2 : 1;

  uint2 yv[NW][2];
  uint4 w[KG ? KG : 1][2][2];
  const int t8 = (FOLD ? t & 1 : t) * 8;
  const bf16* b0 = (const bf16*)g.b + (size_t)max(item.id, 0) * g.N * R + t8;
  const auto load_b = [&](int c, int k0, uint4 (&v)[2][2]) {
    const bf16* b = b0 + (size_t)c * R + k0;
    const bool in = rank > k0 + t8;                           // something of this lane's piece is there
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int j = 2 * hf + m;                             // column 4 g + j
        v[m][hf] = in && c + j < c_end ? load16(b + j * R) : zero4();
      }
  };
  const auto load_all_b = [&](int c) {
    if (KG) {
#pragma unroll
      for (int k = 0; k < KG; ++k) load_b(c, k * 32, w[k]);
    }
  };
  const auto load_y = [&](int c) {
    if (!g.vec || c + 4 > c_end) return;
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = tok0 + j * 8 + 2 * t + i;
        if (tok < item.count) yv[j][i] = *reinterpret_cast<const uint2*>(y + y_at[tok] + c);
      }
  };
  int c0 = c_first + cw * 32;
  if (g.constant && there) load_all_b(c0 + 4 * gq);
  mi_pdl_wait();
  if (!there) return;
  if (!g.constant) load_all_b(c0 + 4 * gq);
  for (int i = tid; i < item.count; i += TILE_THREADS) {
    y_at[i] = rows[i] * g.ldy;
    out_at[i] = rows[i] * g.ldo;
  }

  if (rank > 0) {
    // The sums over all of K, scaled, as two bfloat16 numbers each; whole groups of 32 k (what no sum stands for is zero).
    const float scale = g.scale ? g.scale[item.id] : 1.f;
    const int r4 = (FOLD ? 16 : (R + 31) / 32 * 32) / 4;
    for (int l = lane; l < np * r4; l += 32) {
      const int p = l >= r4, r = (l - p * r4) * 4;
      const float* from = g.h + (part + p) * R + r;
      float4 s[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) s[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll NT == 1 ? 8 : 1
      for (int k = 0; k < g.ks; ++k)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const int tok = warp + u * TILE_WARPS;
          if (tok < item.count && r < rank) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(from + ((size_t)k * g.M + rows[tok]) * PR));
            s[u].x += v.x;
            s[u].y += v.y;
            s[u].z += v.z;
            s[u].w += v.w;
          }
        }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float f[4] = {s[u].x, s[u].y, s[u].z, s[u].w};
        bf16 hi[4], lo[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) split_bf16(r + q < rank ? f[q] * scale : 0.f, hi[q], lo[q]);
        bf16* to = h + (p * 2 * TOK + warp + u * TILE_WARPS) * stride + r;
        *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(hi);
        *reinterpret_cast<uint2*>(to + (FOLD ? 16 : TOK * stride)) = *reinterpret_cast<uint2*>(lo);
      }
    }
  }
  __syncthreads();
  load_y(c0 + 4 * gq);

  const bf16* h0 = h + (tok0 + gq) * stride + t * 8;
  const int second = g.pairs ? 2 * TOK * stride : 0;          // the columns 2 i + 1 of pairs have sums of their own
  for (; c0 < c_end; c0 += CW * 32) {
    const int c = c0 + 4 * gq;
    float acc[2][NW][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    const auto group = [&](int k0, uint4 (&v)[2][2]) {
      const int n = rank - k0 - t8;
      if (n < 8 && n > 0) {                                   // what lies behind the rank
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) v[m][hf] = first_of(v[m][hf], n);
      }
      __syncwarp();
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const bf16* hp = h0 + k0 + (m ? second : 0);
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          mma_k32(acc[m][j], v[m][0], v[m][1], load16(hp + j * 8 * stride));
          if (!FOLD) mma_k32(acc[m][j], v[m][0], v[m][1], load16(hp + (TOK + j * 8) * stride));
        }
      }
    };
    if (KG) {
#pragma unroll
      for (int k = 0; k < KG; ++k)
        if (k * 32 < rank) group(k * 32, w[k]);
    } else {
      for (int k0 = 0; k0 < rank; k0 += 32) {
        load_b(c, k0, w[0]);
        group(k0, w[0]);
      }
    }
    uint2 yc[NW][2];
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) yc[j][i] = yv[j][i];
    if (c0 + CW * 32 < c_end) {
      load_all_b(c + CW * 32);
      load_y(c + CW * 32);
    }
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int tok = tok0 + j * 8 + 2 * t + i;
        if (tok >= item.count) continue;
        bf16* op = out + out_at[tok] + c;
        const float d[4] = {acc[0][j][i], acc[1][j][i], acc[0][j][2 + i], acc[1][j][2 + i]};
        if (g.vec && c + 4 <= c_end) {
          Vec4<bf16> v;
          v.v = yc[j][i];
          if (rank > 0) {
            float f[4];
            v.get(f);
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] += d[q];
            v.set(f);
          }
          v.store(op);
        } else {
          const bf16* yp = y + y_at[tok] + c;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (c + q < c_end) op[q] = rank > 0 ? __float2bfloat16_rn(__bfloat162float(yp[q]) + d[q]) : yp[q];
        }
      }
  }
}

// ---- the plan: rows in the order of their adapters, and items of up to 64 of them

#define PLAN_THREADS 1024
#define PLAN_MAX_ADAPTERS 4096

__global__ void __launch_bounds__(PLAN_THREADS)
adapter_plan_kernel(const int* ids, int M, int n, int* order, int4* items, int max_items) {
  mi_pdl_enter();
  extern __shared__ int plan_smem[];
  int* count = plan_smem;                  // [n + 1] rows of each adapter, the last: rows without one
  int* next = count + n + 1;               // [n + 1] where the next row of each goes
  __shared__ int warp_rows[32], warp_items[32], carry[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= n; i += PLAN_THREADS) count[i] = 0;
  if (tid < 2) carry[tid] = 0;
  __syncthreads();
  const auto bucket = [&](int i) {
    const int id = ids[i];
    return id >= 0 && id < n ? id : n;
  };
  for (int i0 = 0; i0 < M; i0 += PLAN_THREADS) {
    const int i = i0 + tid, b = i < M ? bucket(i) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, b);
    if (b >= 0 && lane == __ffs(same) - 1) atomicAdd(&count[b], __popc(same));
  }
  __syncthreads();
  // first rows and first items, from running sums over the adapters
  for (int i0 = 0; i0 <= n; i0 += PLAN_THREADS) {
    const int i = i0 + tid, rows = i <= n ? count[i] : 0, mine = (rows + MAX_ROWS - 1) / MAX_ROWS;
    int r = rows, m = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) {
        r += a;
        m += b;
      }
    }
    if (lane == 31) {
      warp_rows[warp] = r;
      warp_items[warp] = m;
    }
    __syncthreads();
    int before_r = carry[0], before_m = carry[1];
    for (int w = 0; w < warp; ++w) {
      before_r += warp_rows[w];
      before_m += warp_items[w];
    }
    const int first = before_r + r - rows, item = before_m + m - mine;
    if (i <= n) next[i] = first;
    for (int k = 0; k < mine; ++k)
      if (item + k < max_items)
        items[item + k] = make_int4(i < n ? i : -1, first + k * MAX_ROWS, min(MAX_ROWS, rows - k * MAX_ROWS), 0);
    __syncthreads();
    if (tid == PLAN_THREADS - 1) {
      carry[0] = before_r + r;
      carry[1] = before_m + m;
    }
    __syncthreads();
  }
  for (int i = carry[1] + tid; i < max_items; i += PLAN_THREADS) items[i] = make_int4(-1, 0, 0, 0);
  // rows into their order (which one of an adapter's rows comes first changes nothing that is computed)
  for (int i0 = 0; i0 < M; i0 += PLAN_THREADS) {
    const int i = i0 + tid, b = i < M ? bucket(i) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, b);
    int at = 0;
    if (b >= 0 && lane == __ffs(same) - 1) at = atomicAdd(&next[b], __popc(same));
    at = __shfl_sync(0xffffffffu, at, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1u));
    if (b >= 0) order[at] = i;
  }
}

static int plan_items(int M, int n) { return M / MAX_ROWS + (M < n + 1 ? M : n + 1); }
extern "C" int mi_adapter_plan_sizes(int M, int n, int* max_items) {
  if (M <= FEW_MAX) {
    *max_items = 0;
    return 0;
  }
  if (n > PLAN_MAX_ADAPTERS) MI_REFUSE("adapter_plan: %d adapters, at most %d with more than %d rows", n, PLAN_MAX_ADAPTERS, FEW_MAX);
  *max_items = plan_items(M, n);
  return 0;
}
extern "C" int mi_adapter_plan(const int* ids, int M, int n, int* order, void* items, cudaStream_t stream) {
  if (M <= FEW_MAX) return 0;
  if (n > PLAN_MAX_ADAPTERS) MI_REFUSE("adapter_plan: %d adapters, at most %d with more than %d rows", n, PLAN_MAX_ADAPTERS, FEW_MAX);
  MI_LAUNCH((adapter_plan_kernel), 1, PLAN_THREADS, (size_t)(n + 1) * 2 * sizeof(int), stream, ids, M, n, order, (int4*)items,
            plan_items(M, n));
  MI_RETURN_LAUNCH_STATUS();
}

static int refused_by_cuda(cudaError_t e) {
  (void)cudaGetLastError();
  snprintf(g_mi_error, sizeof(g_mi_error), "CUDA: %s", cudaGetErrorString(e));
  return (int)e;
}

// Dynamic shared memory that takes a block over 48 KB (with what the kernel has besides) is allowed once per kernel and device.
template <typename K>
static cudaError_t allow_smem(K kernel, size_t bytes, size_t* allowed) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || bytes <= 40 * 1024 || bytes <= allowed[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) allowed[dev] = bytes;
  return e;
}

template <int NT>
static cudaError_t launch_tiles(const AdapterArgs& g0, int max_items, cudaStream_t stream) {
  AdapterArgs g = g0;
  constexpr int KW = NT == 1 ? TILE_WARPS : TILE_WARPS / 2, TOK = 8 * NT;
  static size_t allowed[4][64];
  const size_t sums_bytes = (size_t)KW * TOK * (SUM_GROUP + 4) * 4;
  cudaError_t e = allow_smem(adapter_sums_kernel<NT>, sums_bytes, allowed[0]);
  if (e != cudaSuccess) return e;
  const int groups = (g.P * g.R + SUM_GROUP - 1) / SUM_GROUP;
  e = MI_LAUNCH((adapter_sums_kernel<NT>), dim3(g.ks, max_items, groups), TILE_THREADS, sums_bytes, stream, g);
  if (e != cudaSuccess) return e;
  const size_t h_bytes = (size_t)(g.pairs ? 2 : 1) * 2 * TOK * h_stride(g.R) * 2;
  const dim3 grid(count_chunks(g, g.span), max_items);
  if (g.R <= 16) return MI_LAUNCH((adapter_add_kernel<NT, 1, true>), grid, TILE_THREADS, h_bytes, stream, g);
  if (g.R <= 32) return MI_LAUNCH((adapter_add_kernel<NT, 1, false>), grid, TILE_THREADS, h_bytes, stream, g);
  if (g.R <= 64) {
    e = allow_smem(adapter_add_kernel<NT, 2, false>, h_bytes, allowed[1]);
    if (e != cudaSuccess) return e;
    return MI_LAUNCH((adapter_add_kernel<NT, 2, false>), grid, TILE_THREADS, h_bytes, stream, g);
  }
  e = allow_smem(adapter_add_kernel<NT, 0, false>, h_bytes, allowed[2]);
  if (e != cudaSuccess) return e;
  return MI_LAUNCH((adapter_add_kernel<NT, 0, false>), grid, TILE_THREADS, h_bytes, stream, g);
}

// Parts of the sum over K: enough blocks for the chip, at least one unit of 32 k for every warp.
static int sum_parts(int M, int n, int K, int P, int R) {
  const int units = (K + 31) / 32, groups = (P * R + SUM_GROUP - 1) / SUM_GROUP;
  const int items = M <= FEW_MAX ? (M < n + 1 + M / 8 ? M : n + 1 + M / 8) : (M + MAX_ROWS - 1) / MAX_ROWS;
  int ks = 2 * 148 / (items * groups);
  const int most = M <= FEW_MAX ? units / TILE_WARPS : units / (TILE_WARPS / 2) / 2;
  ks = ks < most ? ks : most;
  return ks < 1 ? 1 : ks > 16 ? 16 : ks;
}

// Whether the tensor-core kernels take a call: rows of x, A and B in pieces of 16 bytes, a plan where there are many rows.
static bool in_pieces(const void* x, long long ldx, const void* a, const void* b, int M, int K, int n, int P, int R, int dtype) {
  return dtype == MI_DTYPE_BF16 && n > 0 && R > 0 && R <= 256 && K > 0 && R % 8 == 0 && K % 8 == 0 && mi_aligned(a, 16) &&
         mi_aligned(b, 16) && mi_aligned(x, 16) && (M == 1 || ldx % 8 == 0) && P * R <= 65535 * SUM_GROUP;
}

// Floats of scratch memory (h) that a call needs.
extern "C" long long mi_adapter_scratch(const void* x, long long ldx, const void* a, const void* b, int M, int K, int n, int P,
                                        int R, int dtype) {
  const long long one = (long long)M * P * R;
  return in_pieces(x, ldx, a, b, M, K, n, P, R, dtype) ? one * sum_parts(M, n, K, P, R) : one;
}

extern "C" int mi_adapter_add(const void* y, long long ldy, const void* x, long long ldx, const void* a, const void* b,
                              void* out, long long ldo, const int* ids, const int* order, const void* items, const float* scale,
                              const int* ranks, float* h, int M, int N, int K, int n, int P, int R, int end0, int end1, int end2,
                              int end3, int pairs, int constant, int dtype, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (P < 1 || P > ADAPTER_MAX_PARTS) MI_REFUSE("adapter_add: %d parts, at most %d", P, ADAPTER_MAX_PARTS);
  AdapterArgs g = {x, ldx, y, ldy, out, ldo, a, b, ids, ranks, scale, h, M, N, K, n, P, R, {end0, end1, end2, end3}, pairs, 0, 0, 1,
                   order, (const int4*)items, constant};
  if (in_pieces(x, ldx, a, b, M, K, n, P, R, dtype) && (M <= FEW_MAX || (order && items))) {
    const int max_items = M <= FEW_MAX ? (M < n + 1 + M / 8 ? M : n + 1 + M / 8) : plan_items(M, n);
    if (max_items > 65535) MI_REFUSE("adapter_add: %d rows with %d adapters", M, n);
    bool starts4 = true;
    for (int p = 0; p + 1 < P && !pairs; ++p) starts4 = starts4 && g.ends[p] % 4 == 0;
    g.vec = starts4 && mi_aligned(y, 8) && mi_aligned(out, 8) && (M == 1 || (ldy % 4 == 0 && ldo % 4 == 0));
    g.ks = sum_parts(M, n, K, P, R);
    // Blocks with many columns look for their rows and sums once for all of them; a few waves of blocks fill the chip.
    g.span = 2048;
    while (g.span > 256 && (long long)max_items * count_chunks(g, g.span) < (M <= FEW_MAX ? 3 : 4) * 148) g.span /= 2;
    const cudaError_t e = M <= FEW_MAX ? launch_tiles<1>(g, max_items, stream) : launch_tiles<8>(g, max_items, stream);
    if (e != cudaSuccess) return refused_by_cuda(e);
    MI_RETURN_LAUNCH_STATUS();
  }
  if (M > 65535) MI_REFUSE("adapter_add: %d rows, at most 65535 of operands that are not in pieces of 16 bytes", M);
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
