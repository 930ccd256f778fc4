// lora.hip - low-rank adapters of many requests beside one shared projection.
//
//   out[m][n] = sum_k x[m][k] w[n][k] + sum_r t[m][r] b[id][n][r] (+ bias[n]) (+ residual[m][n])
//   t[m][r]   = scale[id] sum_k x[m][k] a[id][g rank + r][k],   id = ids[m / rows_per_id],   g = n / (N / groups)
//
// ids outside [0, adapters) mean "no adapter" for their rows.  `groups` low-rank pairs stand side by side along N: the fused
// q|k|v projection (layers/SpatialTransformer.py:62-64) has one pair for each of its three parts.
//
// t is rounded to 16 bits, as the matrix cores take it: half a step of t, weighted like the other products' factors; every sum is
// fp32 and the result is rounded once.  It is computed by a launch of its own (lora_shrink_kernel: reads x once more, 2 m k bytes)
// or, where that is cheaper, by the kernel that uses it.  Device times below: MI355X, fp16, operands from HBM.
//   - up to 64 rows (lora_rows_kernel; one token of each request): the product is a stream over w beside the b rows of each request.
//     Bound by the chain of memory latencies behind one another (launch, ids, rows, join).  1 row, 1024 x 1024: 5.6 us with t in
//     the block; 64 rows of 64 adapters of rank 32, 1024 -> 4096: 5.3 us for t and 10.9 for the product, which reads 26 MB at 2.4 TB/s.
//   - many rows, whole tiles of one request (lora_gemm_kernel, MIXED = false): the adapters are more K.  Ranks up to 32: t is a
//     by-product of the same K-loop (one launch).  Larger: behind the K-tiles of (x, w) come tiles of (t, b) through the same ring
//     and MFMAs.  18432 x 640 -> 1920, 3 groups of rank 8: 65 us, 710 TFLOP/s (a library's product alone: 64); MFMAs are busy a third
//     of the time, the 71 MB that leave at the blocks' ends and 10 K-steps a block cost the rest.  18432 x 320 -> 320: 13.3 us.
//     2304 x 1280 -> 1280, rank 64: 5.9 us for t, 18.7 us (424 TFLOP/s; a library's product alone 14.3): 32 x 32 wave tiles read a fragment
//     for each MFMA, 2.8 blocks to a CU, waves wait a third of the time (larger tiles: fewer blocks than CUs; measured 20 - 21 us).
//   - many rows of small requests (MIXED = true): the same with tiles over rows in the order of their adapters.  1155 rows, 5
//     adapters of rank 128, 1024 -> 1024: 10.6 us for t and the order, 13.0 for the product.
#include "common.h"
#include <atomic>
#include <type_traits>

__device__ __attribute__((aligned(16))) unsigned g_lora_zero16[4] = {0u, 0u, 0u, 0u};

struct LoraParams {
  const u16 *x, *w;
  u16* out;
  int ldx, ldw, ldo, M, N, K, nk;
  const float* bias;
  const u16* residual;
  int ldr;
  const u16 *la, *lb;
  const float* scale;
  const int* ids;
  int adapters, rank, groups, rpi;
  float inv_rpi;
  u16* t;  // [M][groups * rank]
  int ldt, tiles_n, per, tpg;  // per = N / groups; request-aligned tiles: tpg column tiles to a group
  int* order;  // mixed tiles: the rows in the order of their adapters, chunk by chunk (nullptr: as they come)
};

__device__ __forceinline__ int lora_id(const LoraParams& p, int row) {
  const int id = p.ids[row / p.rpi];
  return id >= 0 && id < p.adapters ? id : -1;
}

// the same for a wave-uniform row below 64: the quotient by a product (its distance from a whole number is at least 1 / 128 where
// it is not 0) and the word through the scalar cache
__device__ __forceinline__ int lora_row_id(const LoraParams& p, int row) {
  const int id = scalar_i32(p.ids + __builtin_amdgcn_readfirstlane((int)((row + 0.5f) * p.inv_rpi)));
  return id < p.adapters ? id : -1;
}

// ---- rows in the order of their adapters.  A tile of 64 consecutive rows of many requests meets most of the adapters, and each costs
// it another K-tile per 64 ranks; ordered, it meets one or two (1155 rows, 5 adapters of rank 128 beside 1024 x 1024: the product 12.6
// us instead of 17.1).  The blocks that compute t leave the order behind: one of them for
// each LORA_CHUNK rows, wave by wave over eight runs of its rows: adapters are counted per run (whole numbers: any order of the
// additions gives the same), summed to starting places, and every row goes to its run's next place.
constexpr int LORA_CHUNK = 4096, LORA_MAX_SORTED = 1023;  // rows of a chunk; adapters counted in the LDS (one more place for "none")
constexpr int LORA_SORT_BYTES = 8 * (LORA_MAX_SORTED + 1) * 4;
__device__ __forceinline__ void lora_sort_rows(const LoraParams& p, int c0, int* place) {  // 512 threads; place: LDS of LORA_SORT_BYTES
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), n = min(LORA_CHUNK, p.M - c0), nk = p.adapters + 1;
  const int run = ((n + 7) / 8 + 63) & ~63, j0 = wv * run, j1 = min(n, j0 + run);  // at most 512 rows
  int* const mine = place + wv * nk;
  for (int i = t; i < 8 * nk; i += 512) place[i] = 0;
  int key[LORA_CHUNK / 512];
#pragma unroll
  for (int u = 0; u < LORA_CHUNK / 512; ++u) {
    const int j = j0 + 64 * u + lane;
    key[u] = -1;
    if (j < j1) {
      const int id = lora_id(p, c0 + j);
      key[u] = id < 0 ? p.adapters : id;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < LORA_CHUNK / 512; ++u)
    if (key[u] >= 0) atomicAdd(&mine[key[u]], 1);
  __syncthreads();
  if (wv == 0) {
    int base = 0;
    for (int i = 0; i < nk; i += 64) {
      int v[8], sum = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        v[w] = i + lane < nk ? place[w * nk + i + lane] : 0;
        sum += v[w];
      }
      int end = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(end, o);
        if (lane >= o) end += up;
      }
      int at = base + end - sum;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (i + lane < nk) place[w * nk + i + lane] = at;
        at += v[w];
      }
      base += __shfl(end, 63);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int u = 0; u < LORA_CHUNK / 512; ++u) {
    int k = -1;
#pragma unroll
    for (int e = 0; e < LORA_CHUNK / 512; ++e) k = e == u ? key[e] : k;
    int rank = 0, count = 0;
    for (unsigned long long todo = __builtin_amdgcn_ballot_w64(k >= 0); todo;) {
      const unsigned long long same = __builtin_amdgcn_ballot_w64(k == __builtin_amdgcn_readlane(k, __builtin_ctzll(todo)));
      if ((same >> lane) & 1) {
        rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        count = __builtin_popcountll(same);
      }
      todo &= ~same;
    }
    if (k >= 0) {
      const int at = mine[k];
      p.order[c0 + at + rank] = c0 + j0 + 64 * u + lane;
      if (rank == 0) mine[k] = at + count;  // behind the others' reading of it: a wave's LDS instructions keep their order
    }
  }
}

// ---- a wave's own panel of LDS: rows of 64 k, moved by DMA 8 rows (1 KB, whole 128-byte lines) an instruction.  Fragments read
// straight from memory (16 rows x 64 B an instruction) ran at a fifth of this rate: 35 MB took 7.5 us.
constexpr int LBK = 64;
__device__ __forceinline__ int lora_off(int row, int chunk) { return row * LBK + ((chunk ^ ((row >> 1) & 7)) << 3); }
// rows [0, 8 N8) x k [k0, k0 + 64) of a panel to LDS byte address `lds`; rows past `rows` and k past K read as zeros
template <int N8>
__device__ __forceinline__ void lora_panel(const u16* base, int ld, int rows, int k0, int K, unsigned lds, int lane) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, DMA_OOB, 0x00020000);
#pragma unroll
  for (int i = 0; i < N8; ++i) {
    const int r = 8 * i + (lane >> 3), k = k0 + ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    dma_buf16(rs, (r < rows) & (k < K) ? 2u * (unsigned)(r * ld + k) : DMA_OOB, 0, lds + i * 1024);
  }
}

// ------------------------------------------------------------------------------------------------------------ t = scale x a^T
// Block: 16 MR rows by 16 NT columns of t; its eight waves take the K-steps of 64 in turn, each in a panel of its own (S steps in
// flight, no barrier), and join in wave order through the LDS.  A block works for ONE adapter: blockIdx.z is the z-th distinct
// one among its rows; every row keeps its own adapter's result, blocks beyond the last one leave.  With p.order the blocks of
// blockIdx.z = 0 put the rows in order instead.
template <int MR, int NT>
struct ShrinkShape {
  static constexpr int S = 9 / (MR + NT) > 0 ? 9 / (MR + NT) : 1, WAVE = S * (MR + NT) * 2048;  // bytes of a wave's panel
  static constexpr int red = MR * NT * 8192, bytes = 8 * WAVE > red ? 8 * WAVE : red;
};
template <int MR, int NT>
__global__ __launch_bounds__(512, 1) void lora_shrink_kernel(const LoraParams p) {
  typedef ShrinkShape<MR, NT> H;
  extern __shared__ __attribute__((aligned(16))) u16 smem[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, lq = lane >> 4;
  const int row0 = blockIdx.x * (16 * MR), n0 = blockIdx.y * (NT * 16), NR = p.ldt;
  int z = blockIdx.z;
  if (p.order) {
    static_assert(LORA_SORT_BYTES <= H::bytes, "the counts in the panels' memory");
    if (z == 0) {
      if (blockIdx.y == 0 && (long long)blockIdx.x * LORA_CHUNK < p.M) lora_sort_rows(p, blockIdx.x * LORA_CHUNK, (int*)smem);
      return;
    }
    --z;
  }
  const int mine = lane < 16 * MR && row0 + lane < p.M ? lora_id(p, row0 + lane) : -1;
  unsigned long long todo = __builtin_amdgcn_ballot_w64(mine >= 0);  // the same in every wave
  int id = 0;
  for (; todo; --z) {
    id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    if (z == 0) break;
    todo &= ~__builtin_amdgcn_ballot_w64(mine == id);
  }
  if (!todo) return;
  const float sc = p.scale[id];
  f32x4 acc[MR][NT];
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const u16* const xb = p.x + (long long)row0 * p.ldx;
  const u16* const ab = p.la + ((long long)id * NR + n0) * p.K;
  const unsigned lds = lds_addr_of(smem) + wv * H::WAVE;
  const u16* const sm = smem + wv * (H::WAVE / 2);
  for (int k1 = wv; k1 < p.nk; k1 += 8 * H::S) {
#pragma unroll
    for (int s = 0; s < H::S; ++s) {
      const int k0 = (k1 + 8 * s) * LBK;  // past the last step: zeros
      lora_panel<2 * MR>(xb, p.ldx, p.M - row0, k0, p.K, lds + s * (MR + NT) * 2048, lane);
      lora_panel<2 * NT>(ab, p.K, NR - n0, k0, p.K, lds + (s * (MR + NT) + MR) * 2048, lane);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int s = 0; s < H::S; ++s)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        hx8 xf[MR], af[NT];
#pragma unroll
        for (int i = 0; i < MR; ++i) xf[i] = *(const hx8*)&sm[s * (MR + NT) * 1024 + lora_off(16 * i + l15, lq + 4 * kk)];
#pragma unroll
        for (int j = 0; j < NT; ++j) af[j] = *(const hx8*)&sm[(s * (MR + NT) + MR) * 1024 + lora_off(16 * j + l15, lq + 4 * kk)];
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = MFMA16(af[j], xf[i], acc[i][j], 0, 0, 0);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the panel is read before the next steps land in it
  }
  __syncthreads();
  float* const red = (float*)smem;  // [wave][tile][4][64]: row 16 i + l15, column 16 j + 4 lq + e
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[((wv * MR * NT + i * NT + j) * 4 + e) * 64 + lane] = acc[i][j][e];
  __syncthreads();
  for (int q = wv; q < MR * NT; q += 8) {
    const int i = q / NT, j = q - i * NT, n = n0 + 16 * j + 4 * lq;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) y[e] += red[((w * MR * NT + q) * 4 + e) * 64 + lane];
      y[e] *= sc;
    }
    const int his = __shfl(mine, 16 * i + l15);
    if (his == id && n < NR) *(uint2*)(p.t + (long long)(row0 + 16 * i + l15) * p.ldt + n) = make_uint2(pack2h(y[0], y[1]), pack2h(y[2], y[3]));
  }
}

// ------------------------------------------------------------------------------------------------------------ up to 64 rows
// Block: 16 columns x all M <= 16 MT rows; its eight waves take the K-steps in turn, as above: w is read once by the whole grid, x
// by every block (L2).  The adapters: four lanes share a (row, column) pair and take the dot product of t[m] and b[id][n], rank
// long, 16 bytes each at a time; the first 32 ranks of both are fetched before the product, behind the first K-steps' DMA.  FUSE: the block computes t of its rows
// itself (m * groups * rank <= 64 dot products of length K, one wave each in turn) instead of reading what an earlier launch left.
template <int MT>
struct RowsShape {
  static constexpr int S = MT == 4 ? 2 : 9 / (MT + 1), WAVE = S * (MT + 1) * 2048, bytes = 8 * WAVE;  // the join needs 8 MT KB of it
};
template <int MT, bool FUSE>
__global__ __launch_bounds__(512, 1) void lora_rows_kernel(const LoraParams p) {
  typedef RowsShape<MT> H;
  constexpr int NP = MT * 16 * 16 / 128;  // (row, column) pairs a group of four lanes finishes
  extern __shared__ __attribute__((aligned(16))) u16 smem[];
  __shared__ float st[FUSE ? 64 : 1];
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), l15 = lane & 15, lq = lane >> 4, n0 = blockIdx.x * 16;
  // pair x of this lane group: column n0 + c, row x * 8 + (t >> 6)
  const int c = (t >> 2) & 15, piece = t & 3, n = n0 + c, nc = min(n, p.N - 1), g = nc / p.per;
  const u16* const wb = p.w + (long long)n0 * p.ldw;
  const unsigned lds = lds_addr_of(smem) + wv * H::WAVE;
  const u16* const sm = smem + wv * (H::WAVE / 2);
  auto stage = [&](int k1) {
#pragma unroll
    for (int s = 0; s < H::S; ++s) {
      const int k0 = (k1 + 8 * s) * LBK;
      lora_panel<2>(wb, p.ldw, p.N - n0, k0, p.K, lds + s * (MT + 1) * 2048, lane);
      lora_panel<2 * MT>(p.x, p.ldx, p.M, k0, p.K, lds + (s * (MT + 1) + 1) * 2048, lane);
    }
  };
  if (wv < p.nk) stage(wv);  // in flight while the ids and the adapters' rows are fetched
  int id[NP];
  uint4 b0[NP], t0[FUSE ? 1 : NP];
#pragma unroll
  for (int x = 0; x < NP; ++x) {
    const int m = 8 * x + wv;
    id[x] = m < p.M ? lora_row_id(p, m) : -1;
  }
#pragma unroll
  for (int x = 0; x < NP; ++x) {
    b0[x] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (!FUSE) t0[x] = b0[x];
    if (id[x] >= 0 && 8 * piece < p.rank) {
      b0[x] = *(const uint4*)(p.lb + ((long long)id[x] * p.N + nc) * p.rank + 8 * piece);
      if constexpr (!FUSE) t0[x] = *(const uint4*)(p.t + (long long)(8 * x + wv) * p.ldt + g * p.rank + 8 * piece);
    }
  }
  if constexpr (FUSE) {
    // only the groups that this block's columns lie in
    const int g0 = n0 / p.per, g1 = min(n0 + 15, p.N - 1) / p.per, ng = (g1 - g0 + 1) * p.rank;
    for (int d = wv; d < p.M * ng; d += 8) {
      const int m = d / ng, r = g0 * p.rank + (d - m * ng), idm = lora_row_id(p, m);
      if (idm < 0) continue;
      const u16 *xr = p.x + (long long)m * p.ldx, *ar = p.la + ((long long)idm * p.ldt + r) * p.K;
      float s = 0.f;
      for (int k = 8 * lane; k < p.K; k += 512) {
        float xv[8], av[8];
        unpack8(*(const uint4*)(xr + k), xv);
        unpack8(*(const uint4*)(ar + k), av);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(xv[e], av[e], s);
      }
      s = wave_sum(s);
      if (lane == 0) st[m * p.ldt + r] = (float)f2h16(s * p.scale[idm]);  // rounded as the stored t is
    }
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k1 = wv; k1 < p.nk;) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int s = 0; s < H::S; ++s)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const hx8 wf = *(const hx8*)&sm[s * (MT + 1) * 1024 + lora_off(l15, lq + 4 * kk)];
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[i] = MFMA16(wf, *(const hx8*)&sm[(s * (MT + 1) + 1) * 1024 + lora_off(16 * i + l15, lq + 4 * kk)], acc[i], 0, 0, 0);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    k1 += 8 * H::S;
    if (k1 < p.nk) stage(k1);
  }
  __syncthreads();
  float* const red = (float*)smem;  // [wave][4 i + e][64]: row 16 i + l15, column 4 lq + e
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[(wv * MT * 4 + 4 * i + e) * 64 + lane] = acc[i][e];
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NP; ++x) {
    const int m = 8 * x + wv;
    if (m >= p.M) break;  // the rows of a wave rise
    float y = 0.f;
    float bv[8], tv[8];
    auto dot = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) y = __builtin_fmaf(tv[e], bv[e], y);
    };
    const int tb = m * p.ldt + g * p.rank;
    if (id[x] >= 0) {
      unpack8(b0[x], bv);  // zeros past the rank
      if constexpr (FUSE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) tv[e] = 8 * piece < p.rank ? st[tb + 8 * piece + e] : 0.f;
      } else {
        unpack8(t0[x], tv);
      }
      dot();
      const u16* br = p.lb + ((long long)id[x] * p.N + nc) * p.rank;
      for (int r = 32 + 8 * piece; r < p.rank; r += 32) {
        unpack8(*(const uint4*)(br + r), bv);
        if constexpr (FUSE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) tv[e] = st[tb + r + e];
        } else {
          unpack8(*(const uint4*)(p.t + tb + r), tv);
        }
        dot();
      }
    }
    // the eight shares of the product: two to each of the four lanes
#pragma unroll
    for (int w = 0; w < 2; ++w) y += red[((2 * piece + w) * MT * 4 + 4 * (m >> 4) + (c & 3)) * 64 + (c >> 2) * 16 + (m & 15)];
    y += __shfl_xor(y, 1);
    y += __shfl_xor(y, 2);
    if (piece == 0 && n < p.N) {
      if (p.bias) y += p.bias[n];
      if (p.residual) y += h2f(p.residual[(long long)m * p.ldr + n]);
      p.out[(long long)m * p.ldo + n] = f2h(y);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ many rows
// 64 lanes x 16 B from 64 addresses to 1 KB of LDS at byte address `lds`; waited for by the loop's own s_waitcnt
__device__ __forceinline__ void lora_dma16(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}

// FR > 0 (ranks up to FR = 16 or 32, MIXED = false): the block computes t of its rows itself.  FR rows of the adapter's a ride along
// with each K-tile and take one more product per 16 rows and step (the two waves that share rows take alternate steps); behind
// the loop t is joined, scaled, rounded and multiplied with b, whose fragments were fetched before it.  One launch and one
// reading of x less, for FR / (BM + BN) more bytes staged.
// MIXED = false: a tile lies inside one request and one group (the grid is laid out by them), so its adapter is one scalar and the
// adapter's K-tiles are strided like the others.  MIXED = true (requests of fewer rows than a tile): tiles of rows in the order of
// their adapters; the first wave lists the distinct ones, and the adapters' K-tiles are gathered piece by piece.
template <int BM, int BN, int WM, int WN, int NSTAGE, bool MIXED, int FR>
__global__ __launch_bounds__(64 * WM * WN, (WM * WN == 4 && NSTAGE * (BM + BN + FR) * LBK * 2 <= 54 * 1024) ? 3 : 2) void lora_gemm_kernel(const LoraParams p) {
  constexpr int NTH = 64 * WM * WN, RP = NTH / 8, TM = BM / WM, TN = BN / WN, MT = TM / 16, NT = TN / 16, PA = BM / RP, PB = BN / RP;
  constexpr int STAGE = (BM + BN + FR) * LBK;
  static_assert(LORA_CHUNK % BM == 0, "a tile inside one chunk");
  static_assert(FR == 0 || (!MIXED && WN == 2 && NSTAGE == 2 && RP == 32), "t in the block: two waves to a row, all DMA landed at every wait");
  static_assert(BM % RP == 0 && BN % RP == 0 && RP % 16 == 0 && NT % 2 == 0, "tile / wave grid mismatch");
  extern __shared__ __attribute__((aligned(16))) u16 smem[];  // the ring; MIXED: then rowid[BM], the list of adapters [BM], its length and the rows [BM]
  int* const rowid = (int*)(smem + NSTAGE * STAGE);
  int* const list = rowid + BM;
  int* const rowmap = list + BM + 1;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), wr = wv / WN, wc = wv % WN, l15 = lane & 15, lq = lane >> 4;
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int mt = __builtin_amdgcn_readfirstlane(bid / p.tiles_n), nt = bid - mt * p.tiles_n;
  const int per = p.per;
  int brow, rend, bcol, cend, g_lo, ng = 1, nids, id0 = -1;
  if constexpr (MIXED) {
    brow = mt * BM; rend = min(brow + BM, p.M); bcol = nt * BN; cend = min(bcol + BN, p.N);
    g_lo = bcol / per; ng = (cend - 1) / per - g_lo + 1;
    if (t < BM) {
      const int r = brow + t < rend ? (p.order ? p.order[brow + t] : brow + t) : -1;
      rowmap[t] = r;
      rowid[t] = r >= 0 ? lora_id(p, r) : -1;
    }
    if (p.order) brow = brow / LORA_CHUNK * LORA_CHUNK;  // the rows' offsets count from here
    __syncthreads();
    if (wv == 0) {
      int n = 0, v[(BM + 63) / 64];
#pragma unroll
      for (int h = 0; h < (BM + 63) / 64; ++h) v[h] = 64 * h + lane < BM ? rowid[64 * h + lane] : -1;
#pragma unroll
      for (int h = 0; h < (BM + 63) / 64; ++h) {
        unsigned long long todo = __builtin_amdgcn_ballot_w64(v[h] >= 0);
        while (todo) {
          const int id = __builtin_amdgcn_readlane(v[h], __builtin_ctzll(todo));
          if (lane == 0) list[n] = id;
          ++n;
          todo &= ~__builtin_amdgcn_ballot_w64(v[h] == id);
#pragma unroll
          for (int g = 0; g < (BM + 63) / 64; ++g)
            if (g > h && v[g] == id) v[g] = -1;
        }
      }
      if (lane == 0) list[BM] = n;
    }
    __syncthreads();
    nids = __builtin_amdgcn_readfirstlane(list[BM]);
  } else {
    const int tm = (p.rpi + BM - 1) / BM;
    const int req = __builtin_amdgcn_readfirstlane(mt / tm);
    brow = req * p.rpi + (mt - req * tm) * BM;
    rend = min(min(brow + BM, (req + 1) * p.rpi), p.M);
    if (brow >= rend) return;  // the last request may be shorter
    g_lo = __builtin_amdgcn_readfirstlane(nt / p.tpg);
    bcol = g_lo * per + (nt - g_lo * p.tpg) * BN;
    cend = min(bcol + BN, (g_lo + 1) * per);
    id0 = scalar_i32(p.ids + req);
    id0 = id0 < p.adapters ? id0 : -1;
    nids = id0 >= 0 ? 1 : 0;
  }

  const int r0 = t >> 3, lchunk = (t & 7) ^ ((r0 >> 1) & 7);
  int arow[PA];  // the rows of x that this thread moves, behind brow (-1: none)
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    if constexpr (MIXED) {
      const int r = rowmap[r0 + RP * i];
      arow[i] = r < 0 ? -1 : r - brow;
    } else {
      arow[i] = brow + r0 + RP * i < rend ? r0 + RP * i : -1;
    }
  }
  const u16* const xa = p.x + (long long)brow * p.ldx;
  const u16* const wb = p.w + (long long)bcol * p.ldw;
  // MIXED = false: the adapter's panels, t of these rows and b of these columns
  const u16* const ta = p.t + (long long)brow * p.ldt + g_lo * p.rank;
  const u16* const lb = p.lb + ((long long)(id0 < 0 ? 0 : id0) * p.N + bcol) * p.rank;
  const unsigned lds0 = lds_addr_of(smem) + wv * 1024;
  const int nslots = nids * ng, r8 = p.rank >> 3, rk = nids ? p.rank : 0;
  const int ntot = p.nk + (FR ? 0 : (nslots * r8 + 7) / 8);
  const u16* const fa = FR ? p.la + ((long long)(id0 < 0 ? 0 : id0) * p.ldt + g_lo * p.rank) * p.K : nullptr;  // the adapter's rows

  // K-tile KT into ring slot SLOT; always PA + PB DMA instructions per wave (past the last tile: zeros), so that the counted waits
  // below hold
  auto stage = [&](int kt, int slot) {
    const unsigned la = lds0 + slot * (STAGE * 2);
    if (!MIXED || kt < p.nk || kt >= ntot) {
      const bool ext = !MIXED && FR == 0 && kt >= p.nk;
      const int k0 = (ext ? kt - p.nk : kt) * LBK, klim = ext ? rk : p.K;
      const int lda = ext ? p.ldt : p.ldx, ldb = ext ? p.rank : p.ldw;
      const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)(ext ? ta : xa), 0, DMA_OOB, 0x00020000);
      const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)(ext ? lb : wb), 0, DMA_OOB, 0x00020000);
      const unsigned v = 2u * (k0 + lchunk * 8);
      const bool in = k0 + lchunk * 8 < klim;
#pragma unroll
      for (int i = 0; i < PA; ++i)
        dma_buf16(ra, in & (arow[i] >= 0) ? v + 2u * (unsigned)(arow[i] * lda) : DMA_OOB, 0, la + i * (RP * LBK * 2));
#pragma unroll
      for (int i = 0; i < PB; ++i)
        dma_buf16(rb, in & (bcol + r0 + RP * i < cend) ? v + 2u * (unsigned)((r0 + RP * i) * ldb) : DMA_OOB, 0, la + (BM * LBK + i * RP * LBK) * 2);
      if constexpr (FR > 0) {
        if (wv < FR / 8)  // a wave moves 8 rows; the others issue one instruction less, and every wait is for all of them
          dma_buf16(__builtin_amdgcn_make_buffer_rsrc((void*)fa, 0, DMA_OOB, 0x00020000), in & (r0 < rk) ? v + 2u * (unsigned)(r0 * p.K) : DMA_OOB, 0,
                    la + (BM + BN) * LBK * 2);
      }
    } else {
      const u16* const zp = (const u16*)g_lora_zero16;
      const int piece = (kt - p.nk) * 8 + lchunk, s = piece / r8, rc = piece - s * r8;
      const bool ok = s < nslots;
      const int si = s / ng, g = g_lo + s - si * ng, id = ok ? list[si] : 0;
      const int c_lo = g * per, c_hi = c_lo + per;
#pragma unroll
      for (int i = 0; i < PA; ++i) {
        const bool okr = ok && arow[i] >= 0 && rowid[r0 + RP * i] == id;
        lora_dma16(okr ? p.t + (long long)(brow + arow[i]) * p.ldt + g * p.rank + rc * 8 : zp, la + i * (RP * LBK * 2));
      }
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const int n = bcol + r0 + RP * i;
        const bool okn = ok && n < cend && n >= c_lo && n < c_hi;
        lora_dma16(okn ? p.lb + ((long long)id * p.N + n) * p.rank + rc * 8 : zp, la + (BM * LBK + i * RP * LBK) * 2);
      }
    }
  };
#define LORA_WAIT(GROUPS)                                                                           \
  {                                                                                                 \
    constexpr int INFLIGHT = (GROUPS) * (PA + PB);                                                  \
    static_assert(INFLIGHT >= 0 && INFLIGHT < 64, "vmcnt is a 6-bit counter");                      \
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(INFLIGHT) : "memory");          \
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the column that this lane's row of product j stands for: the products 2 i and 2 i + 1 share 32 columns in fours, so that a lane
  // ends up with eight neighbouring ones (a pair of 16-column products would need an exchange between lanes: 3 us of 70)
  auto col = [&](int j) { return 32 * (j >> 1) + 8 * (l15 >> 2) + 4 * (j & 1) + (l15 & 3); };
  constexpr int FT = FR / 16;
  f32x4 tacc[FT ? FT : 1][MT];
  hx8 bf[FT ? NT : 1];
  if constexpr (FR > 0) {
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int i = 0; i < MT; ++i) tacc[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT; ++j) {  // b of this wave's columns, ranks 8 lq .. 8 lq + 7
      const int c = wc * TN + col(j);
      bf[j] = *(const hx8*)(8 * lq < rk && bcol + c < cend ? lb + (long long)c * p.rank + 8 * lq : (const u16*)g_lora_zero16);
    }
  }
  // t: this wave's share of a K-tile (step kk = wc), from the x fragments it has at hand
  auto tmfma = [&](const hx8 (&af)[MT], int slot, int kk) {
    if constexpr (FR > 0) {
      const u16* cF = smem + slot * STAGE + (BM + BN) * LBK;
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        const hx8 ff = *(const hx8*)&cF[lora_off(16 * f + l15, lq + 4 * kk)];
#pragma unroll
        for (int i = 0; i < MT; ++i) tacc[f][i] = MFMA16(ff, af[i], tacc[f][i], 0, 0, 0);
      }
    }
  };
  auto frags = [&](hx8 (&af)[MT], hx8 (&wf)[NT], int slot, int kk) {
    const u16* cA = smem + slot * STAGE;
    const u16* cB = cA + BM * LBK;
#pragma unroll
    for (int i = 0; i < MT; ++i) af[i] = *(const hx8*)&cA[lora_off(wr * TM + i * 16 + l15, lq + 4 * kk)];
#pragma unroll
    for (int j = 0; j < NT; ++j) wf[j] = *(const hx8*)&cB[lora_off(wc * TN + col(j), lq + 4 * kk)];
  };
  auto mfma = [&](const hx8 (&af)[MT], const hx8 (&wf)[NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = MFMA16(wf[j], af[i], acc[i][j], 0, 0, 0);
  };
  // one copy of the staging code for the prologue and one for the loop: a cold block first has to fetch its instructions (with the
  // prologue unrolled the 18432 x 640 x 1920 product took 80 instead of 69 us)
#pragma unroll 1
  for (int s = 0; s < NSTAGE; ++s) stage(s, s);
  hx8 af0[MT], wf0[NT], af1[MT], wf1[NT];
  LORA_WAIT(NSTAGE - 1);
  frags(af0, wf0, 0, 0);
  // the fragments a K-tile starts with are read at the end of the one before, under its last products.  The empty statement keeps
  // the compiler from merging that read with this one into a read at the head of the loop, where its latency shows
#define LORA_PIN() asm volatile("" ::: "memory")
  LORA_PIN();
  int slot = 0;
#pragma unroll 1
  for (int kt = 0; kt < ntot; ++kt) {
    const int nslot = slot + 1 == NSTAGE ? 0 : slot + 1;
    frags(af1, wf1, slot, 1);
    if (FR > 0) {
      if (wc == 0) tmfma(af0, slot, 0);
      else tmfma(af1, slot, 1);
    }
    mfma(af0, wf0);
    LORA_WAIT(NSTAGE - 2);
    stage(kt + NSTAGE, slot);
    frags(af0, wf0, nslot, 0);
    LORA_PIN();
    mfma(af1, wf1);
    slot = nslot;
  }
#undef LORA_PIN
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the trailing DMAs land before the LDS goes to another block
#undef LORA_WAIT
  if constexpr (FR > 0) {
    if (nids) {  // join t of the two waves that share these rows, in the ring's memory: [wc][f][row][rank], 20 floats to a row
      float* const tp = (float*)smem;
      static_assert(2 * FT * BM * 20 * 4 <= NSTAGE * STAGE * 2, "t in the ring");
      __syncthreads();
#pragma unroll
      for (int f = 0; f < FT; ++f)
#pragma unroll
        for (int i = 0; i < MT; ++i) *(f32x4*)&tp[((wc * FT + f) * BM + wr * TM + i * 16 + l15) * 20 + 4 * lq] = tacc[f][i];
      __syncthreads();
      const float sc = p.scale[id0];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        hx8 tf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // ranks 8 lq + 4 h ..
          const int f = FT == 2 ? lq >> 1 : 0, rr = 8 * (lq & 1) + 4 * h;
          const float* q = &tp[(f * BM + wr * TM + i * 16 + l15) * 20 + rr];
          const f32x4 t0 = *(const f32x4*)q, t1 = *(const f32x4*)(q + FT * BM * 20);
#pragma unroll
          for (int e = 0; e < 4; ++e) tf[4 * h + e] = f2h16((t0[e] + t1[e]) * sc);
        }
        if (FT == 1 && lq >= 2) {
#pragma unroll
          for (int e = 0; e < 8; ++e) tf[e] = (h16)0.f;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = MFMA16(bf[j], tf, acc[i][j], 0, 0, 0);
      }
    }
  }
  // A projection without a residual goes to an attention, which reads it once: past the L2, which keeps the operands (with that
  // attention, 96 x 96 to_q 26.3 -> 24.0 us, 48 x 48 q|k|v 219 -> 214).  One that joins the residual stream is what the next product
  // reads over and over: 9216 x 1280 -> 1280 -> 1280 takes 100 us, past the L2 107; 18432 x 320 -> 320 -> 2560 68, 70.  (Two copies of the
  // code: the compiler joins two stores that differ in nothing else.)
  auto finish = [&](auto with_residual) {
    constexpr bool RES = decltype(with_residual)::value;
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      const int n = bcol + wc * TN + 16 * j + 8 * lq;
      const bool okn = n < cend;
      f32x4 b0 = {0.f, 0.f, 0.f, 0.f}, b1 = b0;
      if (p.bias && okn) {
        b0 = *(const f32x4*)(p.bias + n);
        b1 = *(const f32x4*)(p.bias + n + 4);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = MIXED ? rowmap[wr * TM + i * 16 + l15] : brow + wr * TM + i * 16 + l15;
        if ((MIXED ? m >= 0 : m < rend) && okn) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = acc[i][j][e];
            y[4 + e] = acc[i][j + 1][e];
          }
          if (p.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[e] += b0[e];
              y[4 + e] += b1[e];
            }
          }
          if constexpr (RES) {
            float r[8];
            unpack8(*(const uint4*)(p.residual + (long long)m * p.ldr + n), r);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += r[e];
          }
          const uint4 o = pack8(y);
          u32x4* const to = (u32x4*)(p.out + (long long)m * p.ldo + n);
          if constexpr (RES) *to = (u32x4){o.x, o.y, o.z, o.w};
          else __builtin_nontemporal_store((u32x4){o.x, o.y, o.z, o.w}, to);
        }
      }
    }
  };
  if (p.residual) finish(std::true_type{});
  else finish(std::false_type{});
}

// ------------------------------------------------------------------------------------------------------------ host
static bool lora_shape_ok(int m, int n, int k, int rank, int groups) {
  // a group's columns are whole 8-column pieces: the kernels' tiles start at its first
  return m > 0 && m < (1 << 30) && n > 0 && n < (1 << 27) && k > 0 && groups > 0 && groups <= 64 && n % groups == 0 && (n / groups) % 8 == 0 && k % 8 == 0 && rank > 0 && rank % 8 == 0 && rank <= 256;
}
// which kernels take a problem; the workspace holds t where a launch hands it to the next
enum { LORA_ROWS_FUSED, LORA_ROWS, LORA_TILES_FUSED, LORA_TILES, LORA_MIXED };
struct LoraPlan { int kind, bm; };
static LoraPlan lora_plan(int m, int n, int rank, int groups, int rpi) {
  if (m <= 16 && m * groups * rank <= 64) return {LORA_ROWS_FUSED, 0};
  if (m <= 64) return {LORA_ROWS, 0};
  LoraPlan pl;
  pl.bm = (long long)((m + 127) / 128) * ((n + 63) / 64) >= 512 ? 128 : 64;
  // a tile inside one request: when padding every request to whole tiles costs at most a quarter of the rows
  const bool aligned = 4ll * ((rpi + pl.bm - 1) / pl.bm) * pl.bm <= 5ll * rpi;
  pl.kind = !aligned ? LORA_MIXED : rank <= 32 ? LORA_TILES_FUSED : LORA_TILES;
  return pl;
}
static bool lora_needs_t(int kind) { return kind != LORA_ROWS_FUSED && kind != LORA_TILES_FUSED; }
static int64_t lora_t_bytes(int m, int groups, int rank) { return (int64_t)m * groups * rank * 2; }  // a multiple of 16

extern "C" int64_t sdmi_lora_gemm_ws_bytes(int m, int n, int k, int rank, int groups, int rows_per_id) {
  if (!lora_shape_ok(m, n, k, rank, groups) || rows_per_id <= 0) return 0;
  const int kind = lora_plan(m, n, rank, groups, min(rows_per_id, m)).kind;
  return !lora_needs_t(kind) ? 0 : lora_t_bytes(m, groups, rank) + (kind == LORA_MIXED ? (int64_t)m * 4 : 0);  // t, then the rows' order
}

// a kernel with more than 64 KB of dynamic LDS: allowed once per device
template <typename F>
static int lora_allow_lds(F* kernel, int bytes, std::atomic<unsigned long long>& done) {
  if (bytes <= 64 * 1024) return SDMI_OK;
  int dev = 0;
  (void)hipGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return SDMI_OK;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) {
    sdmi_set_error("lora_gemm: %d bytes of LDS refused: %s", bytes, hipGetErrorString(e));
    return SDMI_ELAUNCH;
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return SDMI_OK;
}

template <int MR, int NT>
static int lora_shrink_launch2(const LoraParams& p, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int TR = 16 * MR, bytes = ShrinkShape<MR, NT>::bytes;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  SDMI_REQUIRE((p.M + TR - 1) / TR < (1 << 23), "lora_gemm: grid too large");  // a launch has fewer than 2^32 threads
  const int rc = lora_allow_lds(lora_shrink_kernel<MR, NT>, bytes, done);
  if (rc != SDMI_OK) return rc;
  const int touched = p.rpi >= TR ? (p.rpi % TR == 0 ? 1 : 2) : min((TR - 1 + p.rpi - 1) / p.rpi + 1, TR);  // requests that TR rows can touch
  hipLaunchKernelGGL((lora_shrink_kernel<MR, NT>), dim3((p.M + TR - 1) / TR, (p.ldt + 16 * NT - 1) / (16 * NT), min(touched, p.adapters) + (p.order ? 1 : 0)), dim3(512), bytes, st, p);
  return sdmi_check_launch("lora_gemm (low-rank factor)");
}
static int lora_shrink_launch(const LoraParams& p, hipStream_t st) {
  // larger blocks share more of each reading of x and a; with few of them smaller ones spread over more of the chip
  const int z = p.rpi >= 64 ? 1 : min(p.adapters, 4);
  if (p.ldt > 32 && (long long)((p.M + 63) / 64) * ((p.ldt + 63) / 64) * z >= 128) return lora_shrink_launch2<4, 4>(p, st);
  if (p.ldt > 16 && (long long)((p.M + 31) / 32) * ((p.ldt + 31) / 32) * z >= 128) return lora_shrink_launch2<2, 2>(p, st);
  return p.ldt > 16 ? lora_shrink_launch2<1, 2>(p, st) : lora_shrink_launch2<1, 1>(p, st);
}

template <int BM, int BN, int WM, int WN, int NSTAGE, bool MIXED, int FR>
static int lora_launch(LoraParams p, hipStream_t st) {
  constexpr int bytes = NSTAGE * (BM + BN + FR) * LBK * 2 + (MIXED ? (3 * BM + 1) * 4 : 0);
  static_assert(bytes <= 80 * 1024, "two blocks to a CU");
  static std::atomic<unsigned long long> done{0};
  const int rc = lora_allow_lds(lora_gemm_kernel<BM, BN, WM, WN, NSTAGE, MIXED, FR>, bytes, done);
  if (rc != SDMI_OK) return rc;
  long long tiles_m;
  if (MIXED) {
    p.tiles_n = (p.N + BN - 1) / BN;
    tiles_m = (p.M + BM - 1) / BM;
  } else {
    p.tpg = (p.per + BN - 1) / BN;
    p.tiles_n = p.groups * p.tpg;
    tiles_m = (long long)((p.M + p.rpi - 1) / p.rpi) * ((p.rpi + BM - 1) / BM);
  }
  SDMI_REQUIRE(tiles_m * p.tiles_n < (1ll << 24), "lora_gemm: grid too large");  // a launch has fewer than 2^32 threads
  hipLaunchKernelGGL((lora_gemm_kernel<BM, BN, WM, WN, NSTAGE, MIXED, FR>), dim3((unsigned)(tiles_m * p.tiles_n)), dim3(64 * WM * WN), bytes, st, p);
  sdmi_note_kernel("%slora_gemm_kernel<%d, %d, %s, %d>", FR ? "" : "lora_shrink_kernel + ", BM, BN, MIXED ? "true" : "false", FR);
  return sdmi_check_launch("lora_gemm");
}
template <int BM, int NSTAGE>
static int lora_tiles_launch(const LoraParams& p, int kind, hipStream_t st) {
  if (kind == LORA_MIXED) return lora_launch<BM, 64, 2, 2, NSTAGE, true, 0>(p, st);
  if (kind == LORA_TILES) return lora_launch<BM, 64, 2, 2, NSTAGE, false, 0>(p, st);
  // 128 x 128 tiles, which move a quarter less, once there are four to a CU: 18432 x 640 -> 1920 68 us against 78, 9216 x 640 -> 1920 38 against
  // 41; with fewer 18432 x 320 -> 320 12.4 against 12.1, 18432 x 320 -> 960 28.7 against 27.8 (but 18432 x 640 -> 896 32.7 against 38.7: K counts too)
  if (BM == 128 && (long long)(p.M / 128) * (p.N / 128) >= 1024)
    return p.rank <= 16 ? lora_launch<BM, BM, 2, 2, 2, false, 16>(p, st) : lora_launch<BM, BM, 2, 2, 2, false, 32>(p, st);
  return p.rank <= 16 ? lora_launch<BM, 64, 2, 2, 2, false, 16>(p, st) : lora_launch<BM, 64, 2, 2, 2, false, 32>(p, st);
}
template <int MT, bool FUSE>
static int lora_rows_launch2(const LoraParams& p, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = lora_allow_lds(lora_rows_kernel<MT, FUSE>, RowsShape<MT>::bytes, done);
  if (rc != SDMI_OK) return rc;
  hipLaunchKernelGGL((lora_rows_kernel<MT, FUSE>), dim3((p.N + 15) / 16), dim3(512), RowsShape<MT>::bytes, st, p);
  sdmi_note_kernel("%slora_rows_kernel<%d, %s>", FUSE ? "" : "lora_shrink_kernel + ", MT, FUSE ? "true" : "false");
  return sdmi_check_launch("lora_gemm (few rows)");
}
static int lora_rows_launch(const LoraParams& p, bool fuse, hipStream_t st) {
  if (fuse) return lora_rows_launch2<1, true>(p, st);
  return p.M <= 16 ? lora_rows_launch2<1, false>(p, st) : p.M <= 32 ? lora_rows_launch2<2, false>(p, st) : lora_rows_launch2<4, false>(p, st);
}

extern "C" int sdmi_lora_gemm(const void* x, int ldx, const void* w, int ldw, void* out, int ldo, int m, int n, int k, const float* bias,
                              const void* residual, int ldr, const void* lora_a, const void* lora_b, const float* lora_scale, int adapters,
                              int rank, int groups, const int32_t* ids, int rows_per_id, uint32_t flags, void* ws, int64_t ws_bytes, void* stream) {
  SDMI_REQUIRE(x && w && out && lora_a && lora_b && lora_scale && ids, "lora_gemm: null pointer");
  SDMI_REQUIRE(lora_shape_ok(m, n, k, rank, groups),
               "lora_gemm: bad shape (m %d; n %d, k %d and the rank %d multiples of 8, rank up to 256; %d groups of a multiple of 8 columns)", m, n, k, rank, groups);
  SDMI_REQUIRE(adapters > 0 && rows_per_id > 0, "lora_gemm: %d adapters, %d rows per id", adapters, rows_per_id);
  SDMI_REQUIRE((flags & ~(SDMI_F_BIAS | SDMI_F_RESIDUAL)) == 0, "lora_gemm: flags other than SDMI_F_BIAS and SDMI_F_RESIDUAL");
  SDMI_REQUIRE(!(flags & SDMI_F_BIAS) || bias, "lora_gemm: SDMI_F_BIAS without bias");
  SDMI_REQUIRE(!(flags & SDMI_F_RESIDUAL) || (residual && ldr % 8 == 0 && ldr >= n), "lora_gemm: SDMI_F_RESIDUAL: null residual or bad stride");
  SDMI_REQUIRE(ldx % 8 == 0 && ldw % 8 == 0 && ldo % 8 == 0 && ldx >= k && ldw >= k && ldo >= n, "lora_gemm: strides");
  SDMI_REQUIRE(ldx < (1 << 22) && ldw < (1 << 22), "lora_gemm: x / w row stride too large");  // 32-bit offsets inside a panel
  SDMI_REQUIRE((((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)lora_a | (uintptr_t)lora_b |
                 ((flags & SDMI_F_RESIDUAL) ? (uintptr_t)residual : 0) | ((flags & SDMI_F_BIAS) ? (uintptr_t)bias : 0)) & 15) == 0 &&
                   (((uintptr_t)lora_scale | (uintptr_t)ids) & 3) == 0,
               "lora_gemm: pointer alignment");
  SDMI_REQUIRE(m > 64 || (n + 15) / 16 < (1 << 23), "lora_gemm: grid too large");  // lora_rows_kernel: a launch has fewer than 2^32 threads
  const int64_t need = sdmi_lora_gemm_ws_bytes(m, n, k, rank, groups, rows_per_id);
  SDMI_REQUIRE(need == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= need), "lora_gemm: workspace of %lld bytes, %lld needed, 16-byte aligned",
               (long long)(ws ? ws_bytes : 0), (long long)need);
  rows_per_id = min(rows_per_id, m);  // one id for all rows
  LoraParams p = {};
  p.x = (const u16*)x; p.w = (const u16*)w; p.out = (u16*)out; p.ldx = ldx; p.ldw = ldw; p.ldo = ldo;
  p.M = m; p.N = n; p.K = k; p.nk = (k + LBK - 1) / LBK;
  p.bias = (flags & SDMI_F_BIAS) ? bias : nullptr;
  p.residual = (flags & SDMI_F_RESIDUAL) ? (const u16*)residual : nullptr;
  p.ldr = ldr;
  p.la = (const u16*)lora_a; p.lb = (const u16*)lora_b; p.scale = lora_scale; p.ids = ids;
  p.adapters = adapters; p.rank = rank; p.groups = groups; p.rpi = rows_per_id; p.inv_rpi = 1.0f / rows_per_id;
  p.t = (u16*)ws; p.ldt = groups * rank; p.per = n / groups;
  hipStream_t st = (hipStream_t)stream;
  const LoraPlan pl = lora_plan(m, n, rank, groups, rows_per_id);
  // offsets inside a chunk are 32 bits
  p.order = pl.kind == LORA_MIXED && adapters <= LORA_MAX_SORTED && ldx < (1 << 18) ? (int*)((char*)ws + lora_t_bytes(m, groups, rank)) : nullptr;
  if (lora_needs_t(pl.kind)) {
    const int rc = lora_shrink_launch(p, st);
    if (rc != SDMI_OK) return rc;
  }
  if (pl.kind == LORA_ROWS_FUSED) return lora_rows_launch(p, true, st);
  if (pl.kind == LORA_ROWS) return lora_rows_launch(p, false, st);
  return pl.bm == 128 ? lora_tiles_launch<128, 2>(p, pl.kind, st) : lora_tiles_launch<64, 3>(p, pl.kind, st);
}

extern "C" int sdmi_lora_gemm_packed(const sdmi_lora_gemm_args* a) {
  SDMI_REQUIRE(a, "lora_gemm: null pointer");
  SDMI_REQUIRE(sdmi_fits_int(a->ldx) && sdmi_fits_int(a->ldw) && sdmi_fits_int(a->ldo) && sdmi_fits_int(a->m) && sdmi_fits_int(a->n) && sdmi_fits_int(a->k) && sdmi_fits_int(a->ldr) &&
                   sdmi_fits_int(a->adapters) && sdmi_fits_int(a->rank) && sdmi_fits_int(a->groups) && sdmi_fits_int(a->rows_per_id) && a->flags >= 0 && a->flags <= 0xffffffffll,
               "lora_gemm: bad shape (a size or row stride past 32 bits)");
  return sdmi_lora_gemm(a->x, (int)a->ldx, a->w, (int)a->ldw, a->out, (int)a->ldo, (int)a->m, (int)a->n, (int)a->k, a->bias, a->residual, (int)a->ldr, a->lora_a, a->lora_b,
                        a->lora_scale, (int)a->adapters, (int)a->rank, (int)a->groups, a->ids, (int)a->rows_per_id, (uint32_t)a->flags, a->ws, a->ws_bytes, a->stream);
}
