// Low-rank adapters of many requests beside a projection that all of them share:
//
//   out[t, c] = y[t, c] + sum_r (s_a (A_a x[t])[p(c), r]) B_a[c, r]        a = ids[t]
//   out[t, c] = y[t, c]                                                    where ids[t] is no adapter
//
// A projection may be several merged along its columns; column c belongs to part p(c), and every part has an A of its own:
// A is [adapters, parts, R, K], B [adapters, N, R].  Parts lie side by side, or (pairs) two of them alternate column by column.
// An adapter's own rank may be below R; what lies behind it is not read.  Sums are fp32.
#include "bulk_copy.cuh"

MI_DEFINE_ERROR_API()
MI_DEFINE_STATUS_API(mi_adapters_status)

#define ADAPTER_MAX_PARTS 4

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
  float* h;                       // [parts of the sum over K][M][P R] the sums of the first product
  bf16* held;                     // [M][P][held_sums] the same over all of K, in bfloat16 (many rows)
  int M, N, K, n, P, R;
  int ends[ADAPTER_MAX_PARTS];    // where each part's columns end (side by side)
  int pairs;
  int vec;                        // 4 columns of y and out are one access
  int span;                       // columns of a block (on CUDA cores)
  int ks;                         // parts of the sum over K
  const int* order;
  const int4* items;              // (and behind the last one: how many there are)
  int max_items, tiles;           // of the plan; of columns in a row
  int constant;                   // no kernel in flight writes A and B
};

// What has to move: the rows of x, y and out once, and A and B of the adapters that are used once; the operations, 2 M R (P K + N), are
// few beside it (an adapter of rank 16 does 16 operations for a byte of its own and row).  So the bytes are the floor, and what
// keeps a call from it are latencies: two products of which the second needs all of the first, hence at least two kernels, and the
// way from the ids to the rows.  Three ways, by rows and types:
//
//   few rows (up to FEW_MAX, bfloat16)   mma.sync, blocks find their rows themselves: 6.4 us for a row of rank 16 at 4096 x 6144
//   many rows (bfloat16)                 a plan, tcgen05: 219 us for 8192 rows of ranks to 64 at 4096 x 28672 (155 at the rate of a copy)
//   float32, and what is not in pieces of 16 bytes   CUDA cores
//
// ---------------------------------------------------------------------------------------------- few rows, bfloat16
//
// Both products run on m16n8k16 with the adapter's rows (of A, then of B) as the 16 rows and tokens as the 8 columns, so that
// one token costs an eighth of a tile and not a sixteenth, and operands go from global memory to registers as they lie: a sum over
// k may take its terms in any order, so lane (g, t) = (lane / 4, lane % 4) loads 16 bytes, k = 8 t .. 8 t + 7, of row g, and
// its first two pairs are what the instruction wants for one step of 16 k, the other two for the next.  The instruction takes 32
// cycles of an SM's quarter on this chip, enough for rows by the dozen, whose time the adapters' bytes make.

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

// A sum of the first product as two bfloat16 numbers, h = hi + lo, both of its sign: hi is h cut off behind 8 bits, lo the rest, rounded.
// What is left is up to 2^-16 of h (a rest below 2^-7 of h's power of two, by half a step of its 8 bits), below what the result's
// own rounding leaves.  The second product takes both; where an element of B is infinite they have to say the same, so that lo is never of
// the other sign, nor zero beside a hi that is not: 2^-18 of it is in its place (a sum below 2^-115 aside, which has none).
__device__ __forceinline__ void split_bf16(float v, bf16& hi, bf16& lo) {
  hi = __float2bfloat16_rz(v);
  const float whole = __bfloat162float(hi), rest = v - whole;
  lo = __float2bfloat16_rn(rest == 0.f || isinf(v) ? whole * 0x1p-18f : rest);
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

// Items are up to 8 rows that share an adapter (or have none).  For up to FEW_MAX rows, one to a thread, every block finds the items in the
// ids; for more, adapter_plan has put the rows in order.  FEW_MAX is what the threads of a block look through at once; more would take them
// several turns, and where it would no longer pay has not been measured.  256 rows without a plan and 257 with one, on tcgen05 (us): 32
// adapters of rank 16 at 4096 x 6144 17 and 36, 4 of them 17 and 21, 32 of rank 64 at 4096 x 28672 43 and 98, 4 of them 33 and 32.

#define TILE_THREADS 256
#define TILE_WARPS (TILE_THREADS / 32)
#define FEW_MAX TILE_THREADS  // rows of a call whose items the blocks find by themselves
#define FEW_ROWS 8            // rows of an item
#define SUM_GROUP 64          // sums of the first product that a block makes
#define SUM_BLOCKS (2 * 148)  // blocks of it that the chip holds
#define MAX_ROWS 128          // rows of an item of a plan
#define TILE_COLS (TILE_WARPS * 32)     // columns that a block adds at a time
#define PLAN_TILES 4          // of those, by a block of a call with a plan

struct Item {
  int id, count;              // adapter (-1: none), rows
};
// What a block knows of a call's rows, in shared memory.
struct Rows {
  int4 ids[FEW_MAX / 4];      // the adapter of each row
  int votes[TILE_WARPS];
  unsigned char before[FEW_MAX], leader[FEW_MAX];     // earlier rows with a row's adapter; the first row of each item
  int of_item[FEW_ROWS];      // the rows of the block's item
};

// The items of a call of up to FEW_MAX rows: rows with one adapter are put together in their order, and items are in the order of
// their first rows.  How many there are.
__device__ __forceinline__ int find_items(const AdapterArgs& g, Rows& s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* ids = reinterpret_cast<int*>(s.ids);
  int id = -2;
  if (tid < g.M) {
    id = __ldcg(g.ids + tid);
    if (id >= g.n || id < -1) id = -1;
  }
  ids[tid] = id;
  __syncthreads();
  int before = 0;
  if (tid < g.M) {
    for (int j = 0; j < tid / 4; ++j) {
      const int4 v = s.ids[j];
      before += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
    }
    for (int j = tid & ~3; j < tid; ++j) before += ids[j] == id;
  }
  s.before[tid] = (unsigned char)before;
  const bool leads = tid < g.M && before % FEW_ROWS == 0;
  const unsigned vote = __ballot_sync(0xffffffffu, leads);
  if (lane == 0) s.votes[warp] = __popc(vote);
  __syncthreads();
  int at = __popc(vote & ((1u << lane) - 1u)), all = 0;
#pragma unroll
  for (int w = 0; w < TILE_WARPS; ++w) {
    const int n = s.votes[w];
    at += w < warp ? n : 0;
    all += n;
  }
  if (leads) s.leader[at] = (unsigned char)tid;
  __syncthreads();
  return all;
}
// Item `index` of them (`items` in all), or of the plan; its rows go to s.of_item.  Count 0: there is no such item.
__device__ __forceinline__ Item get_item(const AdapterArgs& g, Rows& s, int index, int items) {
  const int tid = threadIdx.x;
  if (g.items) {
    constexpr int subs = MAX_ROWS / FEW_ROWS;
    const int4 v = __ldcg(g.items + index / subs);
    const int first = index % subs * FEW_ROWS, count = max(0, min(FEW_ROWS, v.z - first));
    if (tid < count) s.of_item[tid] = __ldcg(g.order + v.y + first + tid);
    __syncthreads();
    return Item{v.x, count};
  }
  if (index >= items) return Item{-1, 0};
  const int* ids = reinterpret_cast<const int*>(s.ids);
  const int leader = s.leader[index], id = ids[leader], at = (int)s.before[tid] - (int)s.before[leader];
  const bool mine = tid < g.M && ids[tid] == id && at >= 0 && at < FEW_ROWS;
  if (mine) s.of_item[at] = tid;
  return Item{id, __syncthreads_count(mine)};
}

__device__ __forceinline__ int rank_of(const AdapterArgs& g, int id) {
  return id < 0 ? 0 : g.ranks ? max(0, min(__ldcg(g.ranks + id), g.R)) : g.R;
}

// Parts of the sum over K, up to `most`: all of them where the chip holds that many blocks, else the fewest waves with the shortest
// ways.  A warp's step is 32 k, the rest of a block's time is about two steps, and every part is a quarter of one to the second product.
// All warps come to the same.
__device__ __forceinline__ int sum_parts(int jobs, int units, int most) {
  if (jobs * most <= SUM_BLOCKS) return most;
  const int lane = threadIdx.x & 31, ks = lane + 1;
  unsigned cost = ~0u;
  if (ks <= most) {
    const int waves = (jobs * ks + SUM_BLOCKS - 1) / SUM_BLOCKS, steps = (units + TILE_WARPS * ks - 1) / (TILE_WARPS * ks);
    cost = (unsigned)min(4ll * waves * (steps + 2) + ks, 0x3ffffffll) << 5 | lane;
  }
  return (int)(__reduce_min_sync(0xffffffffu, cost) & 31u) + 1;
}

// The first product: a job is SUM_GROUP sums of an item over a share of K.  The block's warps cut the share between them, their sums meet in
// shared memory and go to h as one part of the sum over K.  Bound by the latency of loads and by the bytes of A.  The number of parts
// follows from the items that there are and not from how many there might be: 160 rows, 32 adapters of rank 64, 4096 x 6144: 26.9 us
// for both kernels, with parts for the most items that 160 rows can make 36.3.
__global__ void __launch_bounds__(TILE_THREADS, 2) adapter_sums_kernel(const AdapterArgs g) {
  constexpr int MT = SUM_GROUP / 16, PAD = SUM_GROUP + 4;
  // The kernel behind this one starts once the ids and operands of both are there; it waits for these sums alone.
  mi_pdl_wait();
  mi_pdl_launch_dependents();
  __shared__ __align__(16) float shares[TILE_WARPS][FEW_ROWS][PAD];
  __shared__ Rows found;
  const int* rows = found.of_item;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  const int items = g.items ? g.max_items : find_items(g, found);
  const int PR = g.P * g.R, groups = (PR + SUM_GROUP - 1) / SUM_GROUP;
  const int units = (g.K + 31) / 32;                          // 32 values of k: 64 bytes of a row
  const int ks = g.items ? g.ks : sum_parts(items * groups, units, g.ks);
  for (int job = blockIdx.x; job < items * groups * ks; job += gridDim.x) {
    const int kp = job / (items * groups), j = job - kp * (items * groups), index = groups == 1 ? j : j / groups;
    const int m0 = (j - index * groups) * SUM_GROUP;
    if (job != (int)blockIdx.x) __syncthreads();              // (what the last job has in shared memory)
    const Item item = get_item(g, found, index, items);
    const int rank = rank_of(g, item.id);
    if (item.count == 0 || rank == 0) continue;
    const int u0 = (int)((long long)units * kp / ks), u1 = (int)((long long)units * (kp + 1) / ks);

    const bool live = gq < item.count;
    const bf16* xr = (const bf16*)g.x + (long long)rows[live ? gq : 0] * g.ldx + t * 8;
    const bf16* ar = (const bf16*)g.a + ((size_t)item.id * PR + m0 + gq) * g.K + t * 8;
    bool have[MT][2], any[MT];                                // sums below the adapter's rank; tiles that have one
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = m0 + m * 16 + hf * 8 + gq;
        have[m][hf] = r < PR && r % g.R < rank;
      }
      any[m] = __any_sync(0xffffffffu, have[m][0] || have[m][1]);
    }
    float acc[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
    // The operands of the next 32 k are loaded before the products of the last ones.
    uint4 xv, av[MT][2];
    const auto load = [&](int u, uint4& xn, uint4 (&an)[MT][2]) {
      const bool in = u < u1 && u * 32 + t * 8 < g.K;
      xn = in && live ? load16(xr + u * 32) : zero4();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          an[m][hf] = in && have[m][hf] ? load16(ar + (size_t)(m * 16 + hf * 8) * g.K + u * 32) : zero4();
    };
    load(u0 + warp, xv, av);
    for (int u = u0 + warp; u < u1; u += TILE_WARPS) {
      uint4 xn, an[MT][2];
      load(u + TILE_WARPS, xn, an);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (any[m]) mma_k32(acc[m], av[m][0], av[m][1], xv);
        av[m][0] = an[m][0];
        av[m][1] = an[m][1];
      }
      xv = xn;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) shares[warp][2 * t + (i & 1)][m * 16 + (i >> 1) * 8 + gq] = acc[m][i];
    __syncthreads();
    float* h = g.h + (size_t)kp * g.M * PR + m0;
    for (int i = tid; i < item.count * (SUM_GROUP / 4); i += TILE_THREADS) {
      const int tok = i / (SUM_GROUP / 4), r = i % (SUM_GROUP / 4) * 4;
      if (m0 + r >= PR) continue;                             // (PR is a multiple of 8)
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < TILE_WARPS; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(&shares[w][tok][r]);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
      *reinterpret_cast<float4*>(h + (size_t)rows[tok] * PR + r) = s;
    }
  }
}

// The second product and the sum with y: a warp takes 32 columns of the item at a time; lane (g, t) ends with columns
// 4 g .. 4 g + 3 of tokens 2 t and 2 t + 1.  B and y of the next columns are loaded between the products and the stores of the last
// ones.
//
// KG: groups of 32 k whose operands are loaded ahead (0: none, ranks above 64).  The rests of the sums ride along: with up to 16 k (FOLD) they
// stand in the place of 16 more, else a product takes four rows and their rests, and an item of more than four rows takes two.
//
// The tiles of all items are shared out over as many blocks as the chip holds, so that hardly one has more than another, whatever the
// items are: 128 rows, 24 adapters, 4096 x 28672: ranks to 64 31.3 us, with blocks of 2048 columns of an item 42.1; rank 16 21.3 and
// 22.6.  BLOCKS of an SM: two, which leaves a thread 128 registers (one row at 4096 x 6144 6.4 us, with three 7.8); three for ranks
// 17 to 32 (96 rows, 32 adapters, 4096 x 28672 30.6 and 32.6).  Columns for two tiles ahead instead of one made no difference.
template <int KG, bool FOLD, int BLOCKS>
__global__ void __launch_bounds__(TILE_THREADS, BLOCKS) adapter_add_kernel(const AdapterArgs g) {
  extern __shared__ __align__(16) unsigned char add_smem[];
  bf16* h = (bf16*)add_smem;                                  // [parts of the block][hi, lo][FEW_ROWS][stride]
  __shared__ Rows found;
  const int* rows = found.of_item;
  mi_pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, t = lane & 3;
  // (the kernel in front was started behind everything that wrote the ids and the operands, and started this one behind that)
  const int items = g.items ? g.max_items : find_items(g, found), R = g.R, PR = g.P * R, stride = h_stride(R), np = g.pairs ? 2 : 1;
  const int ks = g.items ? g.ks : sum_parts(items * ((PR + SUM_GROUP - 1) / SUM_GROUP), (g.K + 31) / 32, g.ks);
  const bf16* y = (const bf16*)g.y;
  bf16* out = (bf16*)g.out;
  int t0, t1;
  if (g.items) {
    t0 = blockIdx.y * g.tiles + min(g.tiles, (int)blockIdx.x * PLAN_TILES);
    t1 = blockIdx.y * g.tiles + min(g.tiles, (int)(blockIdx.x + 1) * PLAN_TILES);
  } else {
    // Whole items in equal pieces, where that makes no block longer by more than a tile, else the same number of tiles for all: another
    // item costs a block a look-up, its sums and a barrier (64 rows, 24 adapters of rank 16 at 4096 x 6144: 11.6 us, 12.5 when blocks
    // take equal numbers always; rank 64 at 4096 x 28672 30.4 and 31.5).
    const long long all = (long long)items * g.tiles;
    const int blocks = (int)gridDim.x, pieces = max(1, min(g.tiles, blocks / items)), longest = (g.tiles + pieces - 1) / pieces;
    if (items <= blocks && longest <= (int)((all + blocks - 1) / blocks) + 1) {
      const int index = (int)blockIdx.x / pieces, piece = (int)blockIdx.x - index * pieces, first = min(index, items) * g.tiles;
      t0 = first + (index < items ? (int)((long long)g.tiles * piece / pieces) : 0);
      t1 = first + (index < items ? (int)((long long)g.tiles * (piece + 1) / pieces) : 0);
    } else {
      t0 = (int)(all * blockIdx.x / blocks);
      t1 = (int)(all * (blockIdx.x + 1) / blocks);
    }
  }

  const int t8 = (FOLD ? t & 1 : t) * 8;
  const bf16* h0 = h + (FOLD ? gq : (gq & 3) + (gq >> 2) * FEW_ROWS) * stride + t * 8;
  const int second = g.pairs ? 2 * FEW_ROWS * stride : 0;     // the columns 2 i + 1 of pairs have sums of their own
  for (int at = t0; at < t1;) {
    // the next stretch of columns of one part of one item
    const int index = at / g.tiles;
    int part, c_first, c_end;
    find_chunk(g, at - index * g.tiles, TILE_COLS, part, c_first, c_end);
    const int tiles = min(t1 - at, (c_end - c_first + TILE_COLS - 1) / TILE_COLS);
    if (at > t0) __syncthreads();                             // (what the last one has in shared memory)
    at += tiles;
    const Item item = get_item(g, found, index, items);
    const int rank = rank_of(g, item.id);
    if (item.count == 0 || (rank == 0 && out == y)) continue;
    c_end = min(c_end, c_first + tiles * TILE_COLS);

    uint2 yv[2];
    uint4 w[KG ? KG : 1][2][2];
    const bf16* b0 = (const bf16*)g.b + (size_t)max(item.id, 0) * g.N * R + t8;
    const auto load_b = [&](int c, int k0, uint4 (&v)[2][2]) {
      const bf16* b = b0 + (size_t)c * R + k0;
      const bool in = rank > k0 + t8;                         // something of this lane's piece is there
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int j = 2 * hf + m;                           // column 4 g + j
          v[m][hf] = in && c + j < c_end ? load16(b + j * R) : zero4();
        }
    };
    const auto load_all_b = [&](int c) {
      if (KG) {
#pragma unroll
        for (int k = 0; k < KG; ++k) load_b(c, k * 32, w[k]);
      }
    };
    int c0 = c_first + warp * 32;
    if (g.constant) load_all_b(c0 + 4 * gq);
    mi_pdl_wait();                                            // (the first time)
    if (!g.constant) load_all_b(c0 + 4 * gq);
    const int mine[2] = {2 * t < item.count ? rows[2 * t] : -1, 2 * t + 1 < item.count ? rows[2 * t + 1] : -1};
    const auto load_y = [&](int c) {
      if (!g.vec || c + 4 > c_end) return;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (mine[i] >= 0) yv[i] = *reinterpret_cast<const uint2*>(y + mine[i] * g.ldy + c);
    };
    load_y(c0 + 4 * gq);

    if (rank > 0) {
      // The sums over all of K, scaled, as two bfloat16 numbers each; whole groups of 32 k (what no sum stands for is zero).
      const float scale = g.scale ? g.scale[item.id] : 1.f;
      const int r4 = (FOLD ? 16 : (R + 31) / 32 * 32) / 4;
      for (int l = lane; l < np * r4; l += 32) {
        const int p = l >= r4, r = (l - p * r4) * 4;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (warp < item.count && r < rank) {
          const float* from = g.h + (size_t)rows[warp] * PR + (part + p) * R + r;
          for (int k0 = 0; k0 < ks; k0 += 8) {                // (eight loads under way, however many there are)
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[k] = k0 + k < ks ? __ldcg(reinterpret_cast<const float4*>(from + (size_t)(k0 + k) * g.M * PR)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              s.x += v[k].x;
              s.y += v[k].y;
              s.z += v[k].z;
              s.w += v[k].w;
            }
          }
        }
        const float f[4] = {s.x, s.y, s.z, s.w};
        bf16 hi[4], lo[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) split_bf16(r + q < rank ? f[q] * scale : 0.f, hi[q], lo[q]);
        bf16* to = h + (p * 2 * FEW_ROWS + warp) * stride + r;
        *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(hi);
        *reinterpret_cast<uint2*>(to + (FOLD ? 16 : FEW_ROWS * stride)) = *reinterpret_cast<uint2*>(lo);
      }
    }
    __syncthreads();

    for (; c0 < c_end; c0 += TILE_COLS) {
      const int c = c0 + 4 * gq;
      float acc[2][4], acc4[2][4];                            // (without FOLD: of rows 0 .. 3 and 4 .. 7)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] = acc4[m][i] = 0.f;
      const auto group = [&](int k0, uint4 (&v)[2][2]) {
        const int n = rank - k0 - t8;
        if (n < 8 && n > 0) {                                 // what lies behind the rank
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) v[m][hf] = first_of(v[m][hf], n);
        }
        __syncwarp();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const bf16* hp = h0 + k0 + (m ? second : 0);
          mma_k32(acc[m], v[m][0], v[m][1], load16(hp));
          if (!FOLD && item.count > 4) mma_k32(acc4[m], v[m][0], v[m][1], load16(hp + 4 * stride));
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
      const uint2 yc[2] = {yv[0], yv[1]};
      if (c0 + TILE_COLS < c_end) {
        load_all_b(c + TILE_COLS);
        load_y(c + TILE_COLS);
      }
      if (!FOLD) {
        // a lane's numbers and their rests', which lane t ^ 2 has: lanes 0 and 1 of four keep rows 0 .. 3, the others 4 .. 7
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, t < 2 ? acc4[m][i] : acc[m][i], 2);
            acc[m][i] = (t < 2 ? acc[m][i] : acc4[m][i]) + other;
          }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (mine[i] < 0) continue;
        bf16* op = out + mine[i] * g.ldo + c;
        const float d[4] = {acc[0][i], acc[1][i], acc[0][2 + i], acc[1][2 + i]};
        if (g.vec && c + 4 <= c_end) {
          Vec4<bf16> v;
          v.v = yc[i];
          if (rank > 0) {
            float f[4];
            v.get(f);
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] += d[q];
            v.set(f);
          }
          v.store(op);
        } else {
          const bf16* yp = y + mine[i] * g.ldy + c;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (c + q < c_end) op[q] = rank > 0 ? __float2bfloat16_rn(__bfloat162float(yp[q]) + d[q]) : yp[q];
        }
      }
    }
  }
  mi_pdl_wait();   // (a block without work: this kernel does not end before the one in front)
}

// ---- the same on CUDA cores: float32, and operands that are not in pieces of 16 bytes
//
// Four values from `k` on, zeros behind `n`.  VEC: they are one access (float32 rows of whole pieces).
template <typename T, bool VEC>
__device__ __forceinline__ float4 four_values(const T* row, int k, int n) {
  if (k >= n) return make_float4(0.f, 0.f, 0.f, 0.f);
  if (VEC && sizeof(T) == 4) return *reinterpret_cast<const float4*>(row + k);
  float4 v;
  v.x = mi_to_float(row[k]);
  v.y = k + 1 < n ? mi_to_float(row[k + 1]) : 0.f;
  v.z = k + 2 < n ? mi_to_float(row[k + 2]) : 0.f;
  v.w = k + 3 < n ? mi_to_float(row[k + 3]) : 0.f;
  return v;
}

// Items of up to eight rows as above, so that what is read of A and B serves all of them; float32 products have no tensor cores that
// keep their bits.  Bound by the loads' latency (one row of rank 16 at 4096 x 6144 8.5 us) and, for many rows, by the CUDA
// cores: 1500 rows 117 us, of which the products at their rate are 3 and the rest is what feeds them.
//
// The first product: a warp makes four sums of an item's up to eight rows over a share of K, its lanes four values of k each; the 32
// totals are shared out over the lanes while they are added up.
#define PLAIN_SUMS 4
#define PLAIN_UNITS 2         // of 128 k in a part of the sum, at least
template <typename T, bool VEC>
__global__ void __launch_bounds__(TILE_THREADS, 3) adapter_sums_plain_kernel(const AdapterArgs g) {
  mi_pdl_wait();
  mi_pdl_launch_dependents();
  __shared__ Rows found;
  const int* rows = found.of_item;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Item item = get_item(g, found, blockIdx.y, g.items ? 0 : find_items(g, found));
  const int rank = rank_of(g, item.id), PR = g.P * g.R, first = (blockIdx.z * TILE_WARPS + warp) * PLAIN_SUMS;
  if (item.count == 0 || rank == 0 || first >= PR) return;
  const int units = (g.K + 127) / 128;
  const int u0 = (int)((long long)units * blockIdx.x / g.ks), u1 = (int)((long long)units * (blockIdx.x + 1) / g.ks);
  const T* x[FEW_ROWS];
#pragma unroll
  for (int t = 0; t < FEW_ROWS; ++t) x[t] = (const T*)g.x + (long long)rows[t < item.count ? t : 0] * g.ldx;
  const T* a = (const T*)g.a + ((size_t)item.id * PR + first) * g.K;
  float acc[PLAIN_SUMS * FEW_ROWS];
#pragma unroll
  for (int i = 0; i < PLAIN_SUMS * FEW_ROWS; ++i) acc[i] = 0.f;
  for (int u = u0; u < u1; ++u) {
    const int k = u * 128 + lane * 4;
    float4 av[PLAIN_SUMS];
#pragma unroll
    for (int j = 0; j < PLAIN_SUMS; ++j)
      av[j] = four_values<T, VEC>(a + (size_t)j * g.K, first + j < PR && (first + j) % g.R < rank ? k : g.K, g.K);
#pragma unroll
    for (int t0 = 0; t0 < FEW_ROWS; t0 += 4) {                // four rows under way at once
      float4 xv[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) xv[t] = four_values<T, VEC>(x[t0 + t], t0 + t < item.count ? k : g.K, g.K);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < PLAIN_SUMS; ++j) {
          float& s = acc[j * FEW_ROWS + t0 + t];
          s = fmaf(xv[t].x, av[j].x, fmaf(xv[t].y, av[j].y, fmaf(xv[t].z, av[j].z, fmaf(xv[t].w, av[j].w, s))));
        }
    }
  }
  // lane l ends with the total of acc[l]
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = upper ? acc[i] : acc[i + o], keep = upper ? acc[i + o] : acc[i];
      acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  const int sum = first + lane / FEW_ROWS, tok = lane % FEW_ROWS;
  if (sum < PR && tok < item.count) g.h[((size_t)blockIdx.x * g.M + rows[tok]) * PR + sum] = acc[0];
}

// The second product and the sum with y: a thread has a column and the item's rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(TILE_THREADS) adapter_add_plain_kernel(const AdapterArgs g) {
  extern __shared__ __align__(16) float plain_h[];            // [parts of the block][R up to 4s][FEW_ROWS]
  __shared__ Rows found;
  const int* rows = found.of_item;
  mi_pdl_launch_dependents();
  const Item item = get_item(g, found, blockIdx.y, g.items ? 0 : find_items(g, found));
  const int rank = rank_of(g, item.id), R = g.R, r4 = (R + 3) & ~3, np = g.pairs ? 2 : 1;
  const T* y = (const T*)g.y;
  T* out = (T*)g.out;
  int part, c_first, c_end;
  const bool there = find_chunk(g, blockIdx.x, g.span, part, c_first, c_end) && item.count > 0 && (rank > 0 || out != y);
  mi_pdl_wait();
  if (!there) return;
  c_end = min(c_end, c_first + g.span);
  if (rank > 0) {
    const float scale = g.scale ? g.scale[item.id] : 1.f;
    for (int i = threadIdx.x; i < np * r4 * FEW_ROWS; i += TILE_THREADS) {
      const int t = i % FEW_ROWS, r = i / FEW_ROWS % r4, p = i / FEW_ROWS / r4;
      float s = 0.f;
      if (t < item.count && r < rank) {
        const float* from = g.h + (size_t)rows[t] * g.P * R + (part + p) * R + r;
#pragma unroll 8
        for (int k = 0; k < g.ks; ++k) s += __ldcg(from + (size_t)k * g.M * g.P * R);
      }
      plain_h[i] = s * scale;
    }
    __syncthreads();
  }
  for (int c = c_first + threadIdx.x; c < c_end; c += TILE_THREADS) {
    if (rank == 0) {
      for (int t = 0; t < item.count; ++t) out[rows[t] * g.ldo + c] = y[rows[t] * g.ldy + c];
      continue;
    }
    float acc[FEW_ROWS], d[FEW_ROWS];
#pragma unroll
    for (int t = 0; t < FEW_ROWS; ++t) {
      acc[t] = t < item.count ? mi_to_float(y[rows[t] * g.ldy + c]) : 0.f;
      d[t] = 0.f;
    }
    const T* b = (const T*)g.b + ((size_t)item.id * g.N + c) * R;
    const float* h = plain_h + (g.pairs ? c & 1 : 0) * r4 * FEW_ROWS;
#pragma unroll 2
    for (int r = 0; r < rank; r += 4) {
      // (a whole piece is loaded, and what lies behind the rank left out)
      const float4 v = VEC ? four_values<T, VEC>(b, r, R) : four_values<T, VEC>(b, r, rank);
      const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (r + q >= rank) break;
        const float4 h0 = *reinterpret_cast<const float4*>(h + (r + q) * FEW_ROWS), h1 = *reinterpret_cast<const float4*>(h + (r + q) * FEW_ROWS + 4);
        d[0] = fmaf(w[q], h0.x, d[0]);
        d[1] = fmaf(w[q], h0.y, d[1]);
        d[2] = fmaf(w[q], h0.z, d[2]);
        d[3] = fmaf(w[q], h0.w, d[3]);
        d[4] = fmaf(w[q], h1.x, d[4]);
        d[5] = fmaf(w[q], h1.y, d[5]);
        d[6] = fmaf(w[q], h1.z, d[6]);
        d[7] = fmaf(w[q], h1.w, d[7]);
      }
    }
#pragma unroll
    for (int t = 0; t < FEW_ROWS; ++t)
      if (t < item.count) out[rows[t] * g.ldo + c] = mi_from_float<T>(acc[t] + d[t]);
  }
}

// ---- many rows: both products on tcgen05, items of up to 128 rows
//
// Operands lie in shared memory as the tensor cores want them: rows of 64 k (128 bytes), 16-byte pieces permuted within a row by the
// row's number modulo 8.  They are brought there piece by piece with cp.async, which gathers the rows of an item from wherever they
// are and leaves zeros for what is not there (rows behind the last, k behind the end or the rank).

#define TC_THREADS 256
#define TC_ROWS 128
#define TC_ATOM (TC_ROWS * 128)      // bytes of 128 rows of 64 k
#define SUMS_MAX_STAGES 4
#define A1_COLS 128                 // columns of a tile of the result
#define A1_MAX_STAGES 4

__device__ __forceinline__ void copy_piece(uint32_t to, const void* from, int bytes) {      // the rest of 16 bytes: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// An operand of rows of 64 k, 128-byte swizzle, groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// bfloat16 x bfloat16 -> fp32, 128 rows by n columns
__device__ __forceinline__ uint32_t product_desc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TC_ROWS >> 4) << 24);
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
               "l"(a), "l"(b), "r"(desc), "r"(accumulate)
               : "memory");
}
// the same with the first operand in tensor memory: row i in lane i, two of k a column
__device__ __forceinline__ void tc_mma_held(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
               "r"(a), "l"(b), "r"(desc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void smem_for_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void tc_load32(uint32_t from, uint32_t (&r)[32]) {      // 32 columns of this thread's row
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(from)
      : "memory");
}
__device__ __forceinline__ void tc_load16(uint32_t from, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(from)
      : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t to, const uint4 (&v)[4]) {      // 16 columns of this thread's row
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(to),
      "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w), "r"(v[2].x), "r"(v[2].y),
      "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w)
      : "memory");
}
__device__ __forceinline__ void tc_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// Tensor memory for a block, by its first warp; the address is in `holder` behind a barrier of the block.  Only then may the next kernel's
// blocks come: one that took the memory while it waits for this kernel would never get an answer.
__device__ __forceinline__ void tc_alloc(uint32_t* holder, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(holder)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tc_free(uint32_t at, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(at), "r"(columns) : "memory");
}

// A stage of the first product: 64 k of 128 rows and of a block's sums
__host__ __device__ inline uint32_t sums_stage_bytes(int PR) { return TC_ATOM + (uint32_t)((PR < 128 ? PR + 15 : 128 + 15) / 16 * 16) * 128; }

struct TcBlock {
  uint64_t bars[SUMS_MAX_STAGES];        // the products that read a stage have ended
  uint32_t tmem;
  int give_up;
  int rows[TC_ROWS];
};

// The item, its rows, barriers and tensor memory; false (for the whole block): nothing to do.
__device__ __forceinline__ bool tc_begin(const AdapterArgs& g, TcBlock& s, int4& item, int& rank) {
  item = __ldcg(g.items + blockIdx.y);
  rank = rank_of(g, item.x);
  if (threadIdx.x < TC_ROWS) s.rows[threadIdx.x] = (int)threadIdx.x < item.z ? __ldcg(g.order + item.y + threadIdx.x) : 0;
  if (threadIdx.x < sizeof(s.bars) / sizeof(s.bars[0])) mbar_init(&s.bars[threadIdx.x], 1);
  if (threadIdx.x == 0) s.give_up = 0;
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  return item.z > 0;
}
__device__ __forceinline__ void tc_ready(TcBlock& s, int columns) {
  if (threadIdx.x < 32) tc_alloc(&s.tmem, columns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  mi_pdl_launch_dependents();
}
// A bounded wait of all threads for the products of a stage; false for all of them when it ran out.
__device__ __forceinline__ bool tc_wait(TcBlock& s, int stage, uint32_t parity) {
  mbar_wait(&s.bars[stage], parity, &s.give_up);
  return __syncthreads_and(!*(volatile int*)&s.give_up);
}

// The first product: up to 128 sums of an item over a share of K, through a ring of stages of 64 k.  Bound by how fast a block
// brings x: 8192 rows of 14336 with rank 16 take 105 us for both products, of which x alone is 36 at the rate of a copy.
template <int STAGES>
__global__ void __launch_bounds__(TC_THREADS) adapter_sums_tc_kernel(const AdapterArgs g) {
  mi_pdl_wait();
  extern __shared__ unsigned char tc_smem[];
  __shared__ TcBlock s;
  const uint32_t base = (smem_u32(tc_smem) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int4 item;
  int rank;
  if (!tc_begin(g, s, item, rank) || rank == 0) return;
  tc_ready(s, 128);
  const int PR = g.P * g.R, m0 = blockIdx.z * 128, sums = min(128, PR - m0), n = (sums + 15) & ~15;
  const int blocks = (g.K + 63) / 64;
  const int u0 = (int)((long long)blocks * blockIdx.x / g.ks), u1 = (int)((long long)blocks * (blockIdx.x + 1) / g.ks);
  const uint32_t stage_bytes = sums_stage_bytes(PR);

  // piece `tid % 8` of four rows of x and of A, 32 rows apart
  const int piece = tid & 7, r0 = tid >> 3;
  const uint32_t place = r0 * 128 + ((piece ^ (r0 & 7)) << 4);
  const bf16 *xr[4], *ar[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = r0 + 32 * j, pr = m0 + row;
    xr[j] = row < item.z ? (const bf16*)g.x + (long long)s.rows[row] * g.ldx + piece * 8 : nullptr;
    ar[j] = row < sums && pr % g.R < rank ? (const bf16*)g.a + ((size_t)item.x * PR + pr) * g.K + piece * 8 : nullptr;
  }
  const auto load = [&](int u) {
    if (u < u1) {
      const uint32_t to = base + (u - u0) % STAGES * stage_bytes + place;
      const bool in = u * 64 + piece * 8 < g.K;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool x_in = in && xr[j], a_in = in && ar[j];
        copy_piece(to + j * 4096, x_in ? xr[j] + u * 64 : (const bf16*)g.x, x_in ? 16 : 0);
        if (r0 + 32 * j < n) copy_piece(to + TC_ATOM + j * 4096, a_in ? ar[j] + u * 64 : (const bf16*)g.a, a_in ? 16 : 0);
      }
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(u0 + i);
  const uint32_t desc = product_desc(n);
  bool ok = true;
  for (int u = u0; u < u1; ++u) {
    copies_wait<STAGES - 2>();
    smem_for_tensor_cores();
    if (__syncthreads_or(*(volatile int*)&s.give_up)) {       // (a wait of the last round ran out)
      ok = false;
      break;
    }
    const int i = u - u0, stage = i % STAGES;
    if (tid == 0) {
      tc_fence_after();
      const uint32_t at = base + stage * stage_bytes;
#pragma unroll
      for (int k = 0; k < 4; ++k) tc_mma(s.tmem, operand_desc(at + k * 32), operand_desc(at + TC_ATOM + k * 32), desc, i > 0 || k > 0);
      tc_commit(&s.bars[stage]);
    }
    // the stage of the products before these is free once they have ended
    if (i > 0) mbar_wait(&s.bars[(i - 1) % STAGES], ((i - 1) / STAGES) & 1, &s.give_up);
    load(u + STAGES - 1);
  }
  copies_wait<0>();
  const int last = u1 - u0 - 1;
  if (ok) ok = tc_wait(s, last % STAGES, (last / STAGES) & 1);
  if (ok) {
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;
    float* h = g.h + ((size_t)blockIdx.x * g.M + s.rows[row]) * PR + m0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int c = (warp >> 2) * 64 + q * 32;
      if (c >= sums) break;                                   // (the whole warp)
      uint32_t v[32];
      tc_load32(s.tmem + ((uint32_t)(warp & 3) << 21) + c, v);
      tc_load_wait();
      if (row < item.z) {
#pragma unroll
        for (int k = 0; k < 32; k += 4)
          if (c + k < sums) *reinterpret_cast<uint4*>(h + c + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (tid < 32) tc_free(s.tmem, 128);
}

// A part's sums for the second product, two bfloat16 numbers each as with few rows: whole groups of 16 k, and behind them their rests.
// In tensor memory they cost no stage of the ring, and the products, twice as many, mostly hide behind the tiles' bytes: 8192 rows of
// rank 64 at 4096 x 28672 219 us, with one number a sum 213, at 4096 x 6144 106 and 104; in a long loop of calls with other inputs each 239
// and 228 (230 with the rests' products left out).
__host__ __device__ inline int padded_rank(int R) { return (R + 15) & ~15; }
__host__ __device__ inline int held_sums(int R) { return 2 * padded_rank(R); }

// The sums over all of K, scaled and split: four sums a thread.  A kernel of its own, since the second product reads them as often as
// an item's tiles are shared out; some 3 us, hidden in part by that kernel's start.
__global__ void __launch_bounds__(256) adapter_held_kernel(const AdapterArgs g) {
  mi_pdl_wait();
  mi_pdl_launch_dependents();
  const int rp = padded_rank(g.R), quarter = rp / 4, per_row = g.P * quarter;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)g.M * per_row) return;
  const int row = (int)(i / per_row), p = (int)(i % per_row) / quarter, r = (int)(i % per_row) % quarter * 4;
  const int id = g.ids[row];
  if (id < 0 || id >= g.n) return;
  const int rank = rank_of(g, id), PR = g.P * g.R;
  const float scale = g.scale ? g.scale[id] : 1.f;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r < rank) {
    const float* from = g.h + (size_t)row * PR + p * g.R + r;
#pragma unroll 4
    for (int k = 0; k < g.ks; ++k) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(from + (size_t)k * g.M * PR));
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
  }
  const float f[4] = {s.x, s.y, s.z, s.w};
  bf16 hi[4], lo[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) split_bf16(r + q < rank ? f[q] * scale : 0.f, hi[q], lo[q]);
  bf16* to = g.held + ((size_t)row * g.P + p) * held_sums(g.R) + r;
  *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(hi);
  *reinterpret_cast<uint2*>(to + rp) = *reinterpret_cast<uint2*>(lo);
}

// Shared memory of the second product: stages of B and of y
__host__ __device__ inline int b_atoms(int R) { return (padded_rank(R) + 63) / 64; }
__host__ __device__ inline int add_stage_bytes(int R) { return b_atoms(R) * TC_ATOM + TC_ROWS * A1_COLS * 2; }

// The second product and the sum with y, in tiles of 128 columns.  One block per SM takes an equal stretch of all items' tiles; its warps
// have parts of their own and meet at mbarriers alone, so that copies, products and sums of different tiles run side by side:
//
//   four copy warps      bring B and y of a tile into a ring of stages, and an item's sums into tensor memory when it begins (a
//                        thread has a row);
//   one thread           issues a tile's products into one of two buffers in tensor memory;
//   eight summing warps  add a buffer to y in shared memory (a thread has a row) and write the result (a lane has pieces of
//                        rows).  y lies in rows of 256 bytes, 16-byte pieces permuted by the row, so that both ways touch all banks.
//
// Bound by memory in long calls: a tile takes 1.6 us of a block, 1.5 us are its bytes at a copy's rate (8192 rows of ranks to 64 at
// 4096 x 28672: 219 us for all kernels, of which this one is some 180), in short ones by the 6 us until the first tile is there.  What a
// warp does for a tile is a chain of latencies, so that a thread's numbers and its y are all asked for at once and a stage is given back
// before the stores (with a sum as one number, 253 us became 213); the first items and their ranks are looked up while tensor memory is allocated
// (2048 rows of rank 16 at 4096 x 4096 33 us become 31).
//
// Copies are cp.async of 16 bytes, a thread's addresses once an item: rows of an item lie anywhere.  (Tensor copies that gather four rows
// at a time have not been tried.)  A copy warp says that a tile is there once its own copies have landed and are visible to the tensor
// cores.
#define A1_SUM_WARPS 8
#define A1_COPY_WARPS 4
#define A1_COPY_THREADS (32 * A1_COPY_WARPS)
#define A1_THREADS (32 * (A1_SUM_WARPS + A1_COPY_WARPS + 1))

#define A1_ITEMS 64                 // items that a block looks up ahead
// Tensor memory: two buffers of a tile's sums, and behind them the first operand, a column for two of a row's sums and rests: at most two
// parts of rank 128.
#define A1_TMEM 512
#define A1_HELD (2 * A1_COLS)

struct AddBlock {
  int4 items[A1_ITEMS];                                     // the first items, their rank instead of the last number
  int n_items;
  uint64_t full[A1_MAX_STAGES], empty[A1_MAX_STAGES];      // a stage is there; the summing warps are through with it
  uint64_t done[2], free_[2];                                // a buffer's products have ended; it has been read
  uint64_t h_free;                                           // the products that read an item's sums have ended
  uint32_t tmem;
  int give_up;
};

// f(tile number of the block, item, rank, whether the item begins, whether it ends, chunk of columns) for a block's tiles in
// order, until f returns false; items of which nothing changes are passed over.
template <typename F>
__device__ __forceinline__ void for_tiles(const AdapterArgs& g, const AddBlock& s, F f) {
  const int per_item = g.tiles;
  const long long all = (long long)s.n_items * per_item;
  const int t0 = (int)(all * blockIdx.x / gridDim.x), t1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
  int count = 0;
  for (int t = t0; t < t1;) {
    const int index = t / per_item, end = min(t1, (index + 1) * per_item);
    const int4 item = index < A1_ITEMS ? s.items[index] : __ldcg(g.items + index);
    const int rank = index < A1_ITEMS ? item.w : rank_of(g, item.x);
    if (rank > 0 || g.out != g.y) {
      for (int u = t; u < end; ++u)
        if (!f(count++, item, rank, u == t, u + 1 == end, u - index * per_item)) return;
    }
    t = end;
  }
}

template <int STAGES, bool PAIRS>
__global__ void __launch_bounds__(A1_THREADS, 1) adapter_add_tc_kernel(const AdapterArgs g) {
  extern __shared__ unsigned char tc_smem[];
  __shared__ AddBlock s;
  // (The kernel in front, which holds the sums, started this one once the first product's had ended: everything that was before that
  // is there, tensor memory is nobody's any more, and the copy warps alone wait, before they take the sums.)
  const uint32_t base = (smem_u32(tc_smem) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, R = g.R;
  const int np = PAIRS ? 2 : 1, rp = padded_rank(R), ba = b_atoms(R);
  const uint32_t stages_at = base, stage_bytes = add_stage_bytes(R);
  if (warp == A1_SUM_WARPS + A1_COPY_WARPS) {
    if (lane == 0) {
      for (int i = 0; i < STAGES; ++i) {
        mbar_init(&s.full[i], A1_COPY_THREADS);
        mbar_init(&s.empty[i], A1_SUM_WARPS);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s.done[i], 1);
        mbar_init(&s.free_[i], A1_SUM_WARPS);
      }
      mbar_init(&s.h_free, 1);
      s.give_up = 0;
      asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    tc_alloc(&s.tmem, A1_TMEM);
  } else if (tid < A1_ITEMS) {
    int4 item = __ldcg(g.items + min(tid, g.max_items - 1));
    if (tid == 0) s.n_items = __ldcg(&g.items[g.max_items].x);
    item.w = rank_of(g, item.x);
    s.items[tid] = item;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  mi_pdl_launch_dependents();
  const uint32_t tmem = s.tmem;
  const bf16* y = (const bf16*)g.y;
  bf16* out = (bf16*)g.out;

  if (warp >= A1_SUM_WARPS && warp < A1_SUM_WARPS + A1_COPY_WARPS) {
    // ---- copies.  Pieces of a row by as many threads, rounded up to a power of two
    constexpr int LAG = STAGES - 2;                           // tiles under way behind the one just asked for
    const int ct = tid - 32 * A1_SUM_WARPS;
    const int b_pieces = rp / 8, b_shift = b_pieces <= 2 ? 1 : b_pieces <= 4 ? 2 : b_pieces <= 8 ? 3 : 4;
    const int bq = ct & ((1 << b_shift) - 1), b_col = ct >> b_shift, b_step = A1_COPY_THREADS >> b_shift;
    const int yq = ct & 15, yr = ct >> 4;                     // piece `yq` of every 8th row
    constexpr int YN = TC_ROWS * 16 / A1_COPY_THREADS;
    const uint32_t y_row = ba * TC_ATOM + yr * 256, y_place[2] = {y_row + ((yq ^ yr) << 4), y_row + ((yq ^ (yr + 8)) << 4)};
    const uint32_t b_place = bq / 8 * TC_ATOM + b_col * 128 + (((bq & 7) ^ (b_col & 7)) << 4);
    const int b_stride = (PAIRS ? 2 : 1) * b_step * R;      // elements between a thread's columns
    const bf16* y_from[YN];
    uint32_t y_in = 0;
    int items = 0, asked = 0, told = 0, last_part = -1;                       // begun so far, of those with an adapter; tiles asked for, and said to be there
    const auto tell = [&](int upto) {
      if (told < upto) smem_for_tensor_cores();
      for (; told < upto; ++told) mbar_arrive(&s.full[told % STAGES]);
    };
    for_tiles(g, s, [&](int j, const int4& item, int rank, bool begins, bool, int chunk) {
      const int stage = j % STAGES;
      const uint32_t to = stages_at + stage * stage_bytes;
      if (begins) {
        y_in = 0;
#pragma unroll
        for (int i = 0; i < YN; ++i) {
          const int row = yr + i * (TC_ROWS / YN);
          if (row < item.z) {
            y_from[i] = y + g.order[item.y + row] * g.ldy + yq * 8;
            y_in |= 1u << i;
          }
        }
      }
      if (j >= STAGES && !__all_sync(0xffffffffu, mbar_wait(&s.empty[stage], (j / STAGES - 1) & 1, &s.give_up))) return false;
      int part, c, c_end;
      find_chunk(g, chunk, A1_COLS, part, c, c_end);
      if (rank > 0 && bq < b_pieces) {
        // rows of B: the tile's columns, of pairs the first ones and then the second ones
        const int there = 2 * max(0, min(8, rank - bq * 8));
        const bf16* b = (const bf16*)g.b + (size_t)item.x * g.N * R + bq * 8;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int first = PAIRS ? c + 2 * b_col + half : c + half * 64 + b_col;
          const bf16* from = b + (size_t)first * R;
          uint32_t at = to + b_place + half * (TC_ATOM / 2);
          if (c + A1_COLS <= c_end && there == 16) {
            for (int col = b_col; col < 64; col += b_step, from += b_stride, at += b_step * 128) copy_piece(at, from, 16);
          } else {
            int column = first;
            for (int col = b_col; col < 64; col += b_step, from += b_stride, at += b_step * 128, column += (PAIRS ? 2 : 1) * b_step) {
              const bool in = there && column < c_end;
              copy_piece(at, in ? from : (const bf16*)g.b, in ? there : 0);
            }
          }
        }
      }
      if (c + yq * 8 < c_end) {
        if (y_in == (1u << YN) - 1u) {
#pragma unroll
          for (int i = 0; i < YN; ++i) copy_piece(to + y_place[i & 1] + i * 2048, y_from[i] + c, 16);
        } else {
#pragma unroll
          for (int i = 0; i < YN; ++i)
            if ((y_in >> i) & 1u) copy_piece(to + y_place[i & 1] + i * 2048, y_from[i] + c, 16);
        }
      }
      copies_commit();
      if ((begins || part != last_part) && rank > 0) {
        last_part = part;
        // the last item's products have to end first, and for that to be told of all their tiles
        copies_wait<1>();
        tell(j);
        if (items > 0 && !__all_sync(0xffffffffu, mbar_wait(&s.h_free, (items - 1) & 1, &s.give_up))) return false;
        if (items++ == 0) mi_pdl_wait();
        tc_fence_after();
        const int row = (warp & 3) * 32 + lane, columns = np * rp;      // (the parts of pairs lie side by side, here and there)
        const uint32_t to_held = tmem + A1_HELD + ((uint32_t)(warp & 3) << 21);
        const uint4* from = reinterpret_cast<const uint4*>(g.held + ((size_t)(row < item.z ? g.order[item.y + row] : 0) * g.P + part) * (2 * rp));
        // A lane's pieces of a row follow one another, so that a sector of L2 serves two of its loads through L1 (past L1, 8192 rows
        // of rank 64 at 4096 x 6144 take 118 us instead of 106).  8 loads under way at once: 16 would not leave registers.
        for (int h0 = 0; h0 < columns; h0 += 32) {
          uint4 v[2][4];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i / 4][i % 4] = row < item.z && h0 + i / 4 * 16 < columns ? from[h0 / 4 + i] : zero4();
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (h0 + i * 16 < columns) tc_store16(to_held + h0 + i * 16, v[i]);
        }
        tc_store_wait();
        tc_fence_before();
      }
      asked = j + 1;
      copies_wait<LAG>();
      tell(asked - LAG);
      return true;
    });
    copies_wait<0>();
    tell(asked);
    mi_pdl_wait();
  } else if (warp == A1_SUM_WARPS + A1_COPY_WARPS) {
    // ---- products
    if (lane == 0) {
      const uint32_t desc = product_desc(PAIRS ? A1_COLS / 2 : A1_COLS);
      for_tiles(g, s, [&](int j, const int4&, int rank, bool, bool ends, int chunk) {
        const int stage = j % STAGES, buf = j & 1;
        if (!mbar_wait(&s.full[stage], (j / STAGES) & 1, &s.give_up)) return false;
        if (j >= 2 && !mbar_wait(&s.free_[buf], (j / 2 - 1) & 1, &s.give_up)) return false;
        tc_fence_after();
        const uint32_t at = stages_at + stage * stage_bytes;
        for (int p = 0; p < np && rank > 0; ++p)
          for (int k = 0; k < rp; k += 16) {
            const uint64_t bd = operand_desc(at + p * 64 * 128 + k / 64 * TC_ATOM + k % 64 * 2);
            for (int lo = 0; lo < 2; ++lo)
              tc_mma_held(tmem + buf * A1_COLS + p * 64, tmem + A1_HELD + p * rp + (k + lo * rp) / 2, bd, desc, k > 0 || lo > 0);
          }
        tc_commit(&s.done[buf]);
        int part, next, c, c_end;
        find_chunk(g, chunk, A1_COLS, part, c, c_end);
        next = part;
        if (!ends) find_chunk(g, chunk + 1, A1_COLS, next, c, c_end);
        if ((ends || next != part) && rank > 0) tc_commit(&s.h_free);
        return true;
      });
    }
    __syncwarp();
  } else {
    // ---- sums: a warp has 32 rows and half of a tile's columns
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21) + (PAIRS ? half * 32 : half * 64);
    const int q0 = lane & 7, r0 = (warp & 3) * 32 + (lane >> 3);       // the result: a piece of every 4th row
    int out_row[8];
    uint32_t out_in = 0;
    for_tiles(g, s, [&](int j, const int4& item, int rank, bool begins, bool, int chunk) {
      const int stage = j % STAGES, buf = j & 1;
      if (begins) {
        out_in = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r0 + 4 * i < item.z) {
            out_row[i] = g.order[item.y + r0 + 4 * i];
            out_in |= 1u << i;
          }
      }
      int part, c, c_end;
      find_chunk(g, chunk, A1_COLS, part, c, c_end);
      const uint32_t y_at = stages_at + stage * stage_bytes + ba * TC_ATOM;
      const bool there = mbar_wait(&s.full[stage], (j / STAGES) & 1, &s.give_up) && mbar_wait(&s.done[buf], (j / 2) & 1, &s.give_up);
      if (!__all_sync(0xffffffffu, there)) return false;
      if (rank > 0) {
        // 32 columns at a time, the next ones on their way meanwhile (a row behind the item's last is added up too, and not written)
        uint32_t v[2][32];
        const uint32_t from = lanes + buf * A1_COLS, y_row = y_at + row * 256, turn = row & 15;
        const auto fetch = [&](int o) {
          tc_load16(from + (PAIRS ? o * 16 : o * 32), v[o]);
          tc_load16(from + (PAIRS ? 64 + o * 16 : o * 32 + 16), v[o] + 16);
        };
        tc_fence_after();
        fetch(0);
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[4 * q]), "=r"(w[4 * q + 1]), "=r"(w[4 * q + 2]), "=r"(w[4 * q + 3])
                         : "r"(y_row + (((half * 8 + o * 4 + q) ^ turn) << 4))
                         : "memory");
          tc_load_wait();
          if (o == 0) {
            fetch(1);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.free_[buf]);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = q * 8 + 2 * e;                    // the pair's first column of the 32
              const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[4 * q + e]));
              const float d0 = __uint_as_float(PAIRS ? v[o][k / 2] : v[o][k]), d1 = __uint_as_float(PAIRS ? v[o][16 + k / 2] : v[o][k + 1]);
              __nv_bfloat162 sum = __floats2bfloat162_rn(f.x + d0, f.y + d1);
              w[4 * q + e] = *reinterpret_cast<uint32_t*>(&sum);
            }
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(y_row + (((half * 8 + o * 4 + q) ^ turn) << 4)), "r"(w[4 * q]),
                         "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                         : "memory");
          }
        }
      } else if (lane == 0) {
        mbar_arrive(&s.free_[buf]);
      }
      __syncwarp();
      const bool mine = c + half * 64 + q0 * 8 < c_end;
      uint4 w[8];
      if (mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((out_in >> i) & 1u) {
            const int r = r0 + 4 * i;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                         : "r"(y_at + r * 256 + (((half * 8 + q0) ^ (r & 15)) << 4))
                         : "memory");
          }
      }
      // (the stage is free once it has been read; the stores follow)
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[stage]);
      if (mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((out_in >> i) & 1u) *reinterpret_cast<uint4*>(out + out_row[i] * g.ldo + (c + half * 64 + q0 * 8)) = w[i];
      }
      return true;
    });
  }
  tc_fence_before();
  __syncthreads();
  if (warp == A1_SUM_WARPS + A1_COPY_WARPS) tc_free(tmem, A1_TMEM);
}

// ---- the plan: rows in the order of their adapters, and items of up to MAX_ROWS of them

#define PLAN_THREADS 1024
#define PLAN_MAX_ADAPTERS 1024

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
  // (rows by the thousand are the usual case: eight loads under way at once)
  const auto for_rows = [&](auto f) {
    for (int i0 = 0; i0 < M; i0 += 8 * PLAN_THREADS) {
      int id[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) id[u] = i0 + u * PLAN_THREADS + tid < M ? ids[i0 + u * PLAN_THREADS + tid] : 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (i0 + u * PLAN_THREADS >= M) break;
        const int i = i0 + u * PLAN_THREADS + tid, b = i >= M ? -1 : id[u] >= 0 && id[u] < n ? id[u] : n;
        // rows side by side are mostly of one request
        int all;
        unsigned same = __match_all_sync(0xffffffffu, b, &all);
        if (!all) same = __match_any_sync(0xffffffffu, b);
        f(i, b, same);
      }
    }
  };
  for_rows([&](int, int b, unsigned same) {
    if (b >= 0 && lane == __ffs(same) - 1) atomicAdd(&count[b], __popc(same));
  });
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
  if (tid == 0) items[max_items] = make_int4(min(carry[1], max_items), 0, 0, 0);
  // rows into their order (which one of an adapter's rows comes first changes nothing that is computed)
  for_rows([&](int i, int b, unsigned same) {
    int at = 0;
    if (b >= 0 && lane == __ffs(same) - 1) at = atomicAdd(&next[b], __popc(same));
    at = __shfl_sync(0xffffffffu, at, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1u));
    if (b >= 0) order[at] = i;
  });
}

static int plan_items(int M, int n) { return M / MAX_ROWS + (M < n + 1 ? M : n + 1); }
extern "C" int mi_adapter_plan_sizes(int M, int n, int* items) {
  if (M <= FEW_MAX) {
    *items = 0;
    return 0;
  }
  if (n > PLAN_MAX_ADAPTERS) MI_REFUSE("adapter_plan: %d adapters, at most %d with more than %d rows", n, PLAN_MAX_ADAPTERS, FEW_MAX);
  *items = plan_items(M, n) + 1;
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

// Dynamic shared memory that takes a block over 48 KB with what the kernel has besides: all that there is is allowed, once per
// kernel and device (so that two threads that come here at once do the same).
template <typename K>
static cudaError_t allow_smem(K kernel, size_t bytes, bool* allowed) {
  if (bytes <= 40 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && allowed[dev])) return e;
  cudaFuncAttributes has;
  e = cudaFuncGetAttributes(&has, kernel);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)has.sharedSizeBytes);
  if (e == cudaSuccess && dev < 64) allowed[dev] = true;
  return e;
}

static cudaError_t launch_few(const AdapterArgs& g, int max_items, cudaStream_t stream) {
  static bool allowed[4][64];
  const int groups = (g.P * g.R + SUM_GROUP - 1) / SUM_GROUP;
  const long long jobs = (long long)max_items * groups * g.ks;
  cudaError_t e = MI_LAUNCH((adapter_sums_kernel), (unsigned)(g.items || jobs < SUM_BLOCKS ? jobs : SUM_BLOCKS), TILE_THREADS, 0, stream, g);
  if (e != cudaSuccess) return e;
  const size_t bytes = (size_t)(g.pairs ? 2 : 1) * 2 * FEW_ROWS * h_stride(g.R) * 2;
  // As many blocks as the chip holds, and no more than there are tiles; or as many as it holds beside the first kernel's, where that makes a
  // block's way a tile longer at most: those are under way when the sums come, the others begin then (8 rows, 8 adapters of rank 16
  // at 4096 x 28672: 9.2 us, with all 296 blocks 11.0).
  const auto run = [&](auto kernel, int blocks, bool* allowed) {
    const cudaError_t e = allow_smem(kernel, bytes, allowed);
    if (e != cudaSuccess) return e;
    const long long most = (long long)max_items * g.tiles, all = blocks * 148, beside = all - (jobs < SUM_BLOCKS ? jobs : SUM_BLOCKS);
    const long long room = beside > 0 && (most + beside - 1) / beside <= (most + all - 1) / all + 1 ? beside : all;
    const dim3 grid = g.items ? dim3((g.tiles + PLAN_TILES - 1) / PLAN_TILES, max_items) : dim3((unsigned)(most < room ? most : room));
    return MI_LAUNCH((kernel), grid, TILE_THREADS, bytes, stream, g);
  };
  if (g.R <= 16) return run(adapter_add_kernel<1, true, 2>, 2, allowed[0]);
  if (g.R <= 32) return run(adapter_add_kernel<1, false, 3>, 3, allowed[1]);
  if (g.R <= 64) return run(adapter_add_kernel<2, false, 2>, 2, allowed[2]);
  return run(adapter_add_kernel<0, false, 2>, 2, allowed[3]);
}

template <typename T, bool VEC>
static cudaError_t launch_plain(const AdapterArgs& g, int max_items, cudaStream_t stream) {
  static bool allowed[64];
  // (also where there is nothing to add: the second kernel looks for its rows ahead of its wait, and may because this one waits)
  const int groups = g.R > 0 ? (g.P * g.R + TILE_WARPS * PLAIN_SUMS - 1) / (TILE_WARPS * PLAIN_SUMS) : 1;
  cudaError_t e = MI_LAUNCH((adapter_sums_plain_kernel<T, VEC>), dim3(g.ks, max_items, groups), TILE_THREADS, 0, stream, g);
  if (e != cudaSuccess) return e;
  const size_t bytes = (size_t)(g.pairs ? 2 : 1) * ((g.R + 3) & ~3) * FEW_ROWS * 4;
  e = allow_smem(adapter_add_plain_kernel<T, VEC>, bytes, allowed);
  if (e != cudaSuccess) return e;
  return MI_LAUNCH((adapter_add_plain_kernel<T, VEC>), dim3(count_chunks(g, g.span), max_items), TILE_THREADS, bytes, stream, g);
}

// Stages that fit: four up to rank 64, three up to 128.
static int add_tc_stages(int R) {      // (of 227 KB 1 is for the alignment and up to 2 are AddBlock's)
  const int n = 224 * 1024 / add_stage_bytes(R);
  return n > A1_MAX_STAGES ? A1_MAX_STAGES : n;
}

static cudaError_t launch_many(const AdapterArgs& g, int max_items, cudaStream_t stream) {
  static bool allowed[6][64];
  const int PR = g.P * g.R;
  const dim3 sums_grid(g.ks, max_items, (PR + 127) / 128);
  // two blocks on an SM: four stages of up to 96 sums, three of more (8192 rows of rank 16 at 14336 x 4096: 105 us, with three 108)
  const int sums_stages = PR <= 96 ? 4 : 3;
  const size_t sums_bytes = (size_t)sums_stages * sums_stage_bytes(PR) + 1024;
  const auto sums = sums_stages == 4 ? adapter_sums_tc_kernel<4> : adapter_sums_tc_kernel<3>;
  cudaError_t e = allow_smem(sums, sums_bytes, allowed[sums_stages == 4 ? 5 : 0]);
  if (e != cudaSuccess) return e;
  e = MI_LAUNCH((sums), sums_grid, TC_THREADS, sums_bytes, stream, g);
  if (e != cudaSuccess) return e;
  const long long quarters = (long long)g.M * g.P * (padded_rank(g.R) / 4);
  e = MI_LAUNCH((adapter_held_kernel), (unsigned)((quarters + 255) / 256), 256, 0, stream, g);
  if (e != cudaSuccess) return e;
  const int stages = add_tc_stages(g.R);
  const size_t bytes = (size_t)stages * add_stage_bytes(g.R) + 1024;
  const long long tiles = (long long)max_items * g.tiles;
  const int grid = tiles < 148 ? (int)tiles : 148;
  const auto run = [&](auto kernel, bool* room) {
    const cudaError_t e = allow_smem(kernel, bytes, room);
    return e != cudaSuccess ? e : MI_LAUNCH((kernel), grid, A1_THREADS, bytes, stream, g);
  };
  if (g.pairs) return stages == 4 ? run(adapter_add_tc_kernel<4, true>, allowed[1]) : run(adapter_add_tc_kernel<3, true>, allowed[2]);
  return stages == 4 ? run(adapter_add_tc_kernel<4, false>, allowed[3]) : run(adapter_add_tc_kernel<3, false>, allowed[4]);
}

// How a call runs, and the scratch memory (h) that it takes.
enum { BY_ELEMENTS, BY_FEW, BY_MANY };
struct Route {
  int way, items, ks;
  long long floats, held_floats;      // of h, and behind it of `held`
};
static Route route_of(const void* y, long long ldy, const void* x, long long ldx, const void* a, const void* b, const void* out,
                      long long ldo, int M, int N, int K, int n, int P, int R, const int* ends, int pairs, int dtype) {
  Route r = {BY_ELEMENTS, 0, 1, (long long)M * P * R, 0};
  r.items = M <= FEW_MAX ? (M < n + 1 + M / FEW_ROWS ? M : n + 1 + M / FEW_ROWS) : plan_items(M, n) * (MAX_ROWS / FEW_ROWS);
  // The tensor-core kernels take rows of x, A and B in pieces of 16 bytes.  mma.sync and CUDA cores, 4 adapters at 4096 x 6144 (us): rank 16,
  // 256 rows 17 and 51; rank 200, 256 rows 48 and 397, 257 over a plan 49 and 375, 2048 272 and 2580.
  if (dtype != MI_DTYPE_BF16 || n <= 0 || R <= 0 || R > 256 || K <= 0 || R % 8 || K % 8 || !mi_aligned(a, 16) ||
      !mi_aligned(b, 16) || !mi_aligned(x, 16) || (M > 1 && ldx % 8)) {
    // Parts of the sum over K follow from K alone, so that float32 rows have the same bits in whatever company.  Rank 16, 4096 x 6144, parts of
    // 256 k and of 512: one row 8.3 and 9.5 us, 1500 rows 117 and 110 (with parts by the number of rows 8.4 and 108).
    const int units = (K + 127) / 128;
    r.ks = units / PLAIN_UNITS;
    r.ks = r.ks < 1 ? 1 : r.ks > 16 ? 16 : r.ks;
    r.floats *= r.ks;
    return r;
  }
  bool whole = N % 8 == 0 && mi_aligned(y, 16) && mi_aligned(out, 16) && (M == 1 || (ldy % 8 == 0 && ldo % 8 == 0));
  for (int p = 0; p + 1 < P && !pairs; ++p) whole = whole && ends[p] % 8 == 0;
  // Over a plan, tcgen05 and mma.sync (us): 4 adapters of rank 16 at 4096 x 6144, 257 rows 20.8 and 19.0, 512 22 and 22, 2048 32 and 51;
  // 32 of them 36.4 and 34.6, 37 and 39, 45 and 69; 4 of rank 64 at 4096 x 28672 32 and 46, 36 and 77, 83 and 251; 32 of them 98 and 100,
  // 101 and 126, 117 and 298.
  if (M > FEW_MAX && whole && R <= 128) {
    r.way = BY_MANY;
    r.items = plan_items(M, n);
    // Parts of the sum over K: enough blocks for the chip, eight stages of 64 k for each (8192 rows of rank 16 at 14336 x 4096: 105 us,
    // with half as many blocks 120, with twice 111)
    const int blocks = (K + 63) / 64, tiles = (M + TC_ROWS - 1) / TC_ROWS * ((P * R + 127) / 128);
    r.ks = 2 * 148 / tiles;
    if (r.ks > blocks / 8) r.ks = blocks / 8;
    r.ks = r.ks < 1 ? 1 : r.ks > 16 ? 16 : r.ks;
    r.held_floats = (long long)M * P * held_sums(R) / 2;
  } else {
    r.way = BY_FEW;
    const int units = (K + 31) / 32, groups = (P * R + SUM_GROUP - 1) / SUM_GROUP;
    // (without a plan the kernels choose, once they know how many items there are)
    r.ks = M <= FEW_MAX ? 16 : SUM_BLOCKS / (r.items * groups);
    if (r.ks > units / (2 * TILE_WARPS)) r.ks = units / (2 * TILE_WARPS);
    r.ks = r.ks < 1 ? 1 : r.ks > 16 ? 16 : r.ks;
  }
  r.floats *= r.ks;
  return r;
}

// The arguments of a call as one block of 64-bit numbers.
struct AdapterCall {
  long long y, ldy, x, ldx, a, b, out, ldo, ids, order, items, scale, ranks, M, N, K, n, P, R, ends[ADAPTER_MAX_PARTS], pairs, constant,
      dtype, unused;
};
static Route route_of(const AdapterCall& c) {
  const int ends[ADAPTER_MAX_PARTS] = {(int)c.ends[0], (int)c.ends[1], (int)c.ends[2], (int)c.ends[3]};
  return route_of((const void*)c.y, c.ldy, (const void*)c.x, c.ldx, (const void*)c.a, (const void*)c.b, (const void*)c.out, c.ldo,
                  (int)c.M, (int)c.N, (int)c.K, (int)c.n, (int)c.P, (int)c.R, ends, (int)c.pairs, (int)c.dtype);
}

// Floats of scratch memory that a call takes.
extern "C" long long mi_adapter_scratch(const AdapterCall* c) {
  const Route r = route_of(*c);
  return r.floats + r.held_floats;
}

extern "C" int mi_adapter_add(const AdapterCall* call, float* h, cudaStream_t stream) {
  const AdapterCall& c = *call;
  const long long most = 0x7fffffff;
  if (c.M > most || c.N > most || c.K > most || c.n > most || c.R > most) MI_REFUSE("adapter_add: sizes beyond 31 bits");
  const int M = (int)c.M, N = (int)c.N, K = (int)c.K, n = (int)c.n, P = (int)c.P, R = (int)c.R, pairs = c.pairs != 0, dtype = (int)c.dtype;
  if (M <= 0 || N <= 0) return 0;
  if (P < 1 || P > ADAPTER_MAX_PARTS) MI_REFUSE("adapter_add: %d parts, at most %d", P, ADAPTER_MAX_PARTS);
  AdapterArgs g = {};
  g.x = (const void*)c.x;
  g.ldx = c.ldx;
  g.y = (const void*)c.y;
  g.ldy = c.ldy;
  g.out = (void*)c.out;
  g.ldo = c.ldo;
  g.a = (const void*)c.a;
  g.b = (const void*)c.b;
  g.ids = (const int*)c.ids;
  g.order = (const int*)c.order;
  g.items = (const int4*)c.items;
  g.ranks = (const int*)c.ranks;
  g.scale = (const float*)c.scale;
  g.h = h;
  g.M = M;
  g.N = N;
  g.K = K;
  g.n = n;
  g.P = P;
  g.R = R;
  for (int p = 0; p < ADAPTER_MAX_PARTS; ++p) g.ends[p] = (int)c.ends[p];
  g.pairs = pairs;
  g.constant = c.constant != 0;
  const Route r = route_of(c);
  if (r.items > 65535) MI_REFUSE("adapter_add: %d rows with %d adapters", M, n);
  if (M > FEW_MAX && !(g.order && g.items)) MI_REFUSE("adapter_add: a plan of %d rows without their order", M);
  if (M <= FEW_MAX) g.items = nullptr;
  g.ks = r.ks;
  if (r.way != BY_ELEMENTS) {
    g.max_items = r.items;
    g.tiles = count_chunks(g, r.way == BY_MANY ? A1_COLS : TILE_COLS);
    if ((long long)r.items * g.tiles > 0x7fffffffLL) MI_REFUSE("adapter_add: %d rows of %d columns", M, N);
    g.held = (bf16*)(h + r.floats);
    bool starts4 = true;
    for (int p = 0; p + 1 < P && !pairs; ++p) starts4 = starts4 && g.ends[p] % 4 == 0;
    g.vec = starts4 && mi_aligned(g.y, 8) && mi_aligned(g.out, 8) && (M == 1 || (g.ldy % 4 == 0 && g.ldo % 4 == 0));
    const cudaError_t e = r.way == BY_MANY ? launch_many(g, r.items, stream) : launch_few(g, r.items, stream);
    if (e != cudaSuccess) return refused_by_cuda(e);
    MI_RETURN_LAUNCH_STATUS();
  }
  // (1500 rows of rank 16 at 4096 x 6144, with parts by the number of rows: 109 us, with half as many blocks 116, with twice 111)
  g.span = 2048;
  while (g.span > 256 && (long long)(M <= FEW_MAX ? r.items : M / FEW_ROWS + n) * count_chunks(g, g.span) < 6 * 148) g.span /= 2;
  if (R > 3000) MI_REFUSE("adapter_add: rank %d, at most 3000", R);
  const cudaError_t e = dtype != MI_DTYPE_F32 ? launch_plain<bf16, false>(g, r.items, stream)
                        : K % 4 || R % 4 || !mi_aligned(g.x, 16) || !mi_aligned(g.a, 16) || !mi_aligned(g.b, 16) || (M > 1 && g.ldx % 4)
                            ? launch_plain<float, false>(g, r.items, stream)
                            : launch_plain<float, true>(g, r.items, stream);
  if (e != cudaSuccess) return refused_by_cuda(e);
  MI_RETURN_LAUNCH_STATUS();
}
