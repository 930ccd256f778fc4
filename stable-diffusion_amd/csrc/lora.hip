// lora.hip - low-rank adapters of many requests beside one shared projection.
//
//   out[m][n] = sum_k x[m][k] w[n][k] + sum_r t[m][r] b[id][n][r] (+ bias[n]) (+ residual[m][n])
//   t[m][r]   = scale[id] sum_k x[m][k] a[id][g rank + r][k],   id = ids[m / rows_per_id],   g = n / (N / groups)
//
// ids outside [0, adapters) mean "no adapter" for their rows.  `groups` low-rank pairs stand side by side along N: the fused
// q|k|v projection (layers/SpatialTransformer.py:62-64) has one pair for each of its three parts.
//
// Two launches: t first (reads x once more: 2 m k bytes, and each adapter's a once per row tile), then the product, in which
// the adapters are more K: behind the K-tiles of (x, w) come tiles whose 16-byte pieces are (t, b) of the (adapter, group)
// pairs that occur in the block's rows and columns, zeros where a row belongs to another adapter.  They pass through the same
// LDS ring and the same MFMAs, so one fp32 accumulator holds the sum and the result is rounded once.  t is rounded to 16 bits
// between the launches, as the matrix cores take it: half a step of t, weighted like the other products' factors.
#include "common.h"

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
  u16* t;   // [M][groups * rank]
  int ldt;
};

__device__ __forceinline__ int lora_id(const LoraParams& p, int row) {
  const int id = p.ids[row / p.rpi];
  return id >= 0 && id < p.adapters ? id : -1;
}

// ------------------------------------------------------------------------------------------------------------ t = scale x a^T
// Block: 16 rows x up to 64 columns of t, K cut over the four waves (32 of it a step), joined in wave order through the LDS.
// Operands come straight from memory in fragment layout (8 consecutive k of one row per lane).  Rows of several adapters: one
// sweep for each, every row keeping its own.
constexpr int SHR_NT = 4;  // 16-column tiles a block computes
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraParams p) {
  __shared__ float red[3][SHR_NT * 4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l15 = lane & 15, lq = lane >> 4;
  const int row = blockIdx.x * 16 + l15, rowc = min(row, p.M - 1), n0 = blockIdx.y * (SHR_NT * 16), NR = p.groups * p.rank;
  const int mine = row < p.M ? lora_id(p, row) : -1;
  const u16* xr = p.x + (long long)rowc * p.ldx;
  unsigned long long todo = __builtin_amdgcn_ballot_w64(mine >= 0);  // the same in every wave
  while (todo) {
    const int id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__builtin_amdgcn_ballot_w64(mine == id);
    const u16* ab = p.la + (long long)id * NR * p.K;
    f32x4 acc[SHR_NT];
#pragma unroll
    for (int j = 0; j < SHR_NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u16* ar[SHR_NT];
#pragma unroll
    for (int j = 0; j < SHR_NT; ++j) ar[j] = ab + (long long)min(n0 + 16 * j + l15, NR - 1) * p.K;
#pragma unroll 4
    for (int kb = wv * 32; kb < p.K; kb += 128) {
      const int k = kb + 8 * lq;
      hx8 xf, af[SHR_NT];
#pragma unroll
      for (int e = 0; e < 8; ++e) xf[e] = (h16)0.f;
#pragma unroll
      for (int j = 0; j < SHR_NT; ++j) af[j] = xf;
      if (k < p.K) {
        xf = *(const hx8*)(xr + k);
#pragma unroll
        for (int j = 0; j < SHR_NT; ++j) af[j] = *(const hx8*)(ar[j] + k);
      }
#pragma unroll
      for (int j = 0; j < SHR_NT; ++j) acc[j] = MFMA16(af[j], xf, acc[j], 0, 0, 0);
    }
    if (wv > 0) {
#pragma unroll
      for (int j = 0; j < SHR_NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wv - 1][4 * j + i][lane] = acc[j][i];
    }
    __syncthreads();
    if (wv == 0 && mine == id) {
      const float sc = p.scale[id];
#pragma unroll
      for (int j = 0; j < SHR_NT; ++j) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (((acc[j][i] + red[0][4 * j + i][lane]) + red[1][4 * j + i][lane]) + red[2][4 * j + i][lane]) * sc;
        const int n = n0 + 16 * j + 4 * lq;
        if (n < NR) *(uint2*)(p.t + (long long)row * p.ldt + n) = make_uint2(pack2h(y[0], y[1]), pack2h(y[2], y[3]));
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------ the product
constexpr int LBK = 64;
__device__ __forceinline__ int lora_off(int row, int chunk) { return row * LBK + ((chunk ^ ((row >> 1) & 7)) << 3); }
// 64 lanes x 16 B from 64 addresses to 1 KB of LDS at byte address `lds`; waited for by the loop's own s_waitcnt
__device__ __forceinline__ void lora_dma16(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}

template <int BM, int BN, int WM, int WN, int NSTAGE>
__global__ __launch_bounds__(64 * WM * WN, 2) void lora_gemm_kernel(const LoraParams p) {
  constexpr int NTH = 64 * WM * WN, RP = NTH / 8, TM = BM / WM, TN = BN / WN, MT = TM / 16, NT = TN / 16, PA = BM / RP, PB = BN / RP;
  constexpr int STAGE = (BM + BN) * LBK;
  static_assert(BM % RP == 0 && BN % RP == 0 && RP % 16 == 0 && BM <= 128, "tile / wave grid mismatch");
  extern __shared__ __attribute__((aligned(16))) u16 smem[];  // the ring, then rowid[BM], the list of adapters [BM] and its length
  int* const rowid = (int*)(smem + NSTAGE * STAGE);
  int* const list = rowid + BM;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, wr = wv / WN, wc = wv % WN, l15 = lane & 15, lq = lane >> 4;
  const int tiles_n = (p.N + BN - 1) / BN, tiles_m = (p.M + BM - 1) / BM;
  const int bid = xcd_remap(blockIdx.x, tiles_m * tiles_n);
  const int brow = bid / tiles_n * BM, bcol = bid % tiles_n * BN;

  const int r0 = t >> 3, lchunk = (t & 7) ^ ((r0 >> 1) & 7), wave_row0 = __builtin_amdgcn_readfirstlane(wv) * 8;
  const __amdgpu_buffer_rsrc_t rsrcA = __builtin_amdgcn_make_buffer_rsrc((void*)(p.x + (long long)brow * p.ldx), 0, DMA_OOB, 0x00020000);
  const __amdgpu_buffer_rsrc_t rsrcB = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + (long long)bcol * p.ldw), 0, DMA_OOB, 0x00020000);
  unsigned a_voff[PA], b_voff[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) a_voff[i] = brow + r0 + RP * i < p.M ? (unsigned)(((r0 + RP * i) * p.ldx + lchunk * 8) * 2) : DMA_OOB;
#pragma unroll
  for (int i = 0; i < PB; ++i) b_voff[i] = bcol + r0 + RP * i < p.N ? (unsigned)(((r0 + RP * i) * p.ldw + lchunk * 8) * 2) : DMA_OOB;
  const unsigned lds0 = lds_addr_of(smem);

  // ---- the adapters of this block's rows.  One request covers them all (the usual case for images): a scalar load.  Else the
  // first wave lists the distinct ones, in the order of their first rows.
  const int last = min(brow + BM, p.M) - 1;
  const bool one = brow / p.rpi == last / p.rpi;
  int id0 = -1, nids;
  if (one) {
    id0 = lora_id(p, brow);
    nids = id0 >= 0 ? 1 : 0;
  } else {
    if (t < BM) rowid[t] = brow + t <= last ? lora_id(p, brow + t) : -1;
    __syncthreads();
    if (wv == 0) {
      int n = 0;
      int v[(BM + 63) / 64];
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
    nids = list[BM];
  }
  const int per = p.N / p.groups;
  const int g_lo = bcol / per, ng = (min(bcol + BN, p.N) - 1) / per - g_lo + 1;
  const int r8 = p.rank >> 3, nslots = nids * ng;
  const int ntot = p.nk + (nslots * r8 + 7) / 8;
  const u16* const zp = (const u16*)g_lora_zero16;

  // K-tile KT into ring slot SLOT; always PA + PB DMA instructions per wave, so that the counted waits below hold
  auto stage = [&](int kt, int slot) {
    const unsigned la = lds0 + (slot * STAGE + wave_row0 * LBK) * 2;
    if (kt < p.nk || kt >= ntot) {
      const bool in = kt * LBK + lchunk * 8 < p.K;
      const int soff = kt * (LBK * 2);
#pragma unroll
      for (int i = 0; i < PA; ++i) dma_buf16(rsrcA, in ? a_voff[i] : DMA_OOB, soff, la + i * (RP * LBK * 2));
#pragma unroll
      for (int i = 0; i < PB; ++i) dma_buf16(rsrcB, in ? b_voff[i] : DMA_OOB, soff, la + (BM * LBK + i * RP * LBK) * 2);
    } else {
      const int piece = (kt - p.nk) * 8 + lchunk, s = piece / r8, rc = piece - s * r8;
      const bool ok = s < nslots;
      const int g = g_lo + s % ng, id = ok ? (one ? id0 : list[s / ng]) : 0;
#pragma unroll
      for (int i = 0; i < PA; ++i) {
        const int r = r0 + RP * i;
        const bool okr = ok && brow + r < p.M && (one || rowid[r] == id);
        lora_dma16(okr ? p.t + (long long)(brow + r) * p.ldt + g * p.rank + rc * 8 : zp, la + i * (RP * LBK * 2));
      }
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const int n = bcol + r0 + RP * i;
        const bool okn = ok && n < p.N && n / per == g;
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
  auto frags = [&](hx8 (&af)[MT], hx8 (&wf)[NT], int slot, int kk) {
    const u16* cA = smem + slot * STAGE;
    const u16* cB = cA + BM * LBK;
#pragma unroll
    for (int i = 0; i < MT; ++i) af[i] = *(const hx8*)&cA[lora_off(wr * TM + i * 16 + l15, lq + 4 * kk)];
#pragma unroll
    for (int j = 0; j < NT; ++j) wf[j] = *(const hx8*)&cB[lora_off(wc * TN + j * 16 + l15, lq + 4 * kk)];
  };
  auto mfma = [&](const hx8 (&af)[MT], const hx8 (&wf)[NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = MFMA16(wf[j], af[i], acc[i][j], 0, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < NSTAGE; ++s) stage(s, s);
  hx8 af0[MT], wf0[NT], af1[MT], wf1[NT];
  LORA_WAIT(NSTAGE - 1);
  frags(af0, wf0, 0, 0);
  int slot = 0;
  for (int kt = 0; kt < ntot; ++kt) {
    const int nslot = slot + 1 == NSTAGE ? 0 : slot + 1;
    frags(af1, wf1, slot, 1);
    mfma(af0, wf0);
    LORA_WAIT(NSTAGE - 2);
    stage(kt + NSTAGE, slot);
    frags(af0, wf0, nslot, 0);
    mfma(af1, wf1);
    slot = nslot;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the trailing DMAs land before the LDS goes to another block
#undef LORA_WAIT
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = brow + wr * TM + i * 16 + l15;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = bcol + wc * TN + j * 16 + 4 * lq;
      if (n >= p.N) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = acc[i][j][e] + (p.bias ? p.bias[n + e] : 0.f);
      if (p.residual) {
        const uint2 rr = *(const uint2*)(p.residual + (long long)m * p.ldr + n);
        float r4[4];
        unpack2(rr.x, r4[0], r4[1]);
        unpack2(rr.y, r4[2], r4[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += r4[e];
      }
      *(uint2*)(p.out + (long long)m * p.ldo + n) = make_uint2(pack2h(y[0], y[1]), pack2h(y[2], y[3]));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ host
static bool lora_shape_ok(int m, int n, int k, int rank, int groups) {
  return m > 0 && n > 0 && k > 0 && groups > 0 && n % groups == 0 && n % 8 == 0 && k % 8 == 0 && rank > 0 && rank % 8 == 0 && rank <= 256 && groups <= 64;
}

extern "C" int64_t sdmi_lora_gemm_ws_bytes(int m, int n, int k, int rank, int groups) {
  return lora_shape_ok(m, n, k, rank, groups) ? (int64_t)m * groups * rank * 2 : 0;
}

template <int BM, int BN, int WM, int WN, int NSTAGE>
static int lora_launch(const LoraParams& p, hipStream_t st) {
  constexpr int bytes = NSTAGE * (BM + BN) * LBK * 2 + (2 * BM + 1) * 4;
  static_assert(bytes <= 64 * 1024, "LDS without an attribute");
  const long long blocks = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  SDMI_REQUIRE(blocks < (1ll << 31), "lora_gemm: grid too large");
  hipLaunchKernelGGL((lora_gemm_kernel<BM, BN, WM, WN, NSTAGE>), dim3((unsigned)blocks), dim3(64 * WM * WN), bytes, st, p);
  sdmi_note_kernel("lora_shrink_kernel + lora_gemm_kernel<%d, %d>", BM, BN);
  return sdmi_check_launch("lora_gemm");
}

extern "C" int sdmi_lora_gemm(const void* x, int ldx, const void* w, int ldw, void* out, int ldo, int m, int n, int k, const float* bias,
                              const void* residual, int ldr, const void* lora_a, const void* lora_b, const float* lora_scale, int adapters,
                              int rank, int groups, const int32_t* ids, int rows_per_id, uint32_t flags, void* ws, int64_t ws_bytes, void* stream) {
  SDMI_REQUIRE(x && w && out && lora_a && lora_b && lora_scale && ids && ws, "lora_gemm: null pointer");
  SDMI_REQUIRE(lora_shape_ok(m, n, k, rank, groups),
               "lora_gemm: bad shape (m %d; n %d, k %d and the rank %d multiples of 8, rank up to 256; %d groups that divide n)", m, n, k, rank, groups);
  SDMI_REQUIRE(adapters > 0 && rows_per_id > 0, "lora_gemm: %d adapters, %d rows per id", adapters, rows_per_id);
  SDMI_REQUIRE((flags & ~(SDMI_F_BIAS | SDMI_F_RESIDUAL)) == 0, "lora_gemm: flags other than SDMI_F_BIAS and SDMI_F_RESIDUAL");
  SDMI_REQUIRE(!(flags & SDMI_F_BIAS) || bias, "lora_gemm: SDMI_F_BIAS without bias");
  SDMI_REQUIRE(!(flags & SDMI_F_RESIDUAL) || (residual && ldr % 8 == 0 && ldr >= n), "lora_gemm: SDMI_F_RESIDUAL: null residual or bad stride");
  SDMI_REQUIRE(ldx % 8 == 0 && ldw % 8 == 0 && ldo % 8 == 0 && ldx >= k && ldw >= k && ldo >= n, "lora_gemm: strides");
  SDMI_REQUIRE(ldx < (1 << 22) && ldw < (1 << 22), "lora_gemm: x / w row stride too large");  // 32-bit offsets inside a panel
  SDMI_REQUIRE((((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)lora_a | (uintptr_t)lora_b | (uintptr_t)ws |
                 ((flags & SDMI_F_RESIDUAL) ? (uintptr_t)residual : 0)) & 15) == 0 &&
                   (((uintptr_t)lora_scale | (uintptr_t)ids | ((flags & SDMI_F_BIAS) ? (uintptr_t)bias : 0)) & 3) == 0,
               "lora_gemm: pointer alignment");
  SDMI_REQUIRE(ws_bytes >= sdmi_lora_gemm_ws_bytes(m, n, k, rank, groups), "lora_gemm: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
               (long long)sdmi_lora_gemm_ws_bytes(m, n, k, rank, groups));
  LoraParams p = {};
  p.x = (const u16*)x; p.w = (const u16*)w; p.out = (u16*)out; p.ldx = ldx; p.ldw = ldw; p.ldo = ldo;
  p.M = m; p.N = n; p.K = k; p.nk = (k + LBK - 1) / LBK;
  p.bias = (flags & SDMI_F_BIAS) ? bias : nullptr;
  p.residual = (flags & SDMI_F_RESIDUAL) ? (const u16*)residual : nullptr;
  p.ldr = ldr;
  p.la = (const u16*)lora_a; p.lb = (const u16*)lora_b; p.scale = lora_scale; p.ids = ids;
  p.adapters = adapters; p.rank = rank; p.groups = groups; p.rpi = rows_per_id;
  p.t = (u16*)ws; p.ldt = groups * rank;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(lora_shrink_kernel, dim3((m + 15) / 16, (groups * rank + 16 * SHR_NT - 1) / (16 * SHR_NT)), dim3(256), 0, st, p);
  int rc = sdmi_check_launch("lora_gemm (low-rank factor)");
  if (rc != SDMI_OK) return rc;
  if ((long long)((m + 127) / 128) * ((n + 63) / 64) >= 512) return lora_launch<128, 64, 2, 2, 2>(p, st);
  return lora_launch<64, 64, 2, 2, 3>(p, st);
}
