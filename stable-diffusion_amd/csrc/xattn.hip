// xattn.hip - cross-attention to encoder states of another length: ragged, shared between samples, with regions.
//
//   o[b][i][h] = sum_j p_ij v[c][j][h'] / sum_j p_ij,   p_ij = [j seen by i] exp(scale q[b][i][h] . k[c][j][h'] - max)
//   c = index[b] (the context of sample b), h' = h * kv_heads / heads, j < lens[c], and with regions
//   (query_regions[b][i] & key_regions[c][j]) != 0.  A row that sees nothing is 0.
//
// The reference has one rectangular case of it (layers/SpatialTransformer.py:70-95: every sample its own context of 77
// tokens, no mask); csrc/attention.hip runs that one.  Here the rows of a kv head's tile are (query, head of the group)
// pairs, so the heads that share keys share their reads, and a batch of samples that share a context reads it through L2.
//
// Mathematics: one pass over the keys with the running maximum m and sum l of the softmax, in base 2: p = 2^((s - m) c), s and m dot
// products of q and k as they are, c = scale * log2(e).  S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: the
// query is on the lane in both, so the statistics are lane-local plus one exchange of the wave's halves, and P leaves the
// first product in the operand layout of the second (k order inside a 16-key step as the accumulator has it; V is read
// through ds_read_b64_tr_b16 in that order).  P is rounded to 16 bits for the matrix cores (half a step of its value);
// S, m, l and O stay in fp32.
//
// What bounds it (MI355X, fp16, device times).  Long states: 9.7 vector instructions beside each MFMA (the exponent's fma and exp2, the
// maximum, the row sum, the packing), MFMAs busy a third of the time - 2 x 10 heads of 64, 2304 rows to 9216 keys 135 us, 803 TFLOP/s; 96 x 96
// rows 301 us, 722; heads of 128 to 4096 keys 124 us, 622; 160: 130 us, 744; 80: 75 us, 645; 256 (one wave to a SIMD): 155 us, 498.  That is
// this loop's form, not the problem's: attn64x2_kernel, for equal lengths and queries that carry log2(e), needs 6.8 and takes 134 and 226
// us for the first two.  The prompt's lengths: the start of a block (Q, the first tile, the store: memory latencies behind one another, two
// to four blocks to a CU to cover them) - 2 x 5 heads, 9216 rows to 77 keys 11.3 us, 2304 rows to 154 keys in regions 14.8 us; 16 x 20 heads,
// 576 rows to 231 shared keys 22.5 us (4.5 blocks of 128 rows, 1.6 rounds of blocks, the last of four tiles on the masked path: 22 vector
// instructions to an MFMA).  One row: the reading of the keys - 320 rows to 9216 keys (755 MB) 138 + 5 us, 5.3 TB/s; 8 x 16 heads of 128 on 4,
// 4096 keys (38 MB where half exist) 13.1 + 4.0 us, half of each block's waves without rows.
#include "common.h"
#include <atomic>

struct XattnParams {
  const u16 *q, *k, *v;
  u16* o;
  long long sq, sk, sv, so;
  int ldq, ldk, ldv, ldo;
  int batch, contexts, heads, kvh, group, dim, nq, nkv, rows, rtiles, splits;  // rows = nq * group: the rows of one kv head
  const int *index, *lens;
  const unsigned *qreg, *kreg;
  long long sqr, skr;
  float c, raise;  // scale * log2(e); XA_RAISE / c
  float* po;    // splits > 1: [row][split][dim] un-normalised partial outputs
  float2* pml;  // [row][split] (m, l)
};

// Start of the running maximum: finite, so that m - m is 0, and so far below every dot product (up to 1e38 in magnitude, scaled too; of
// fp16 they are at most 256 * 65504^2) that the first one raises it: `raise` is at most 1e38.
constexpr float XA_LOWEST = -3.4e38f, XA_RAISE_MAX = 1e38f;

// LDS images of a tile are linear in 16-byte pieces (a wave's DMA writes 1 KB in lane order), DP / 8 pieces to a row; the piece
// that lies at position c of row r is c ^ xa_kx(r) (K) or c ^ xa_vx(r) (V), applied on the source side.  K fragments: 8
// consecutive rows at one logical piece have to fall on 8 different quarters of the 64 banks; V: a transposed read takes 4
// rows x 64 B, which have to fall on 4 different quarters.  Rows of 64, 192 or 320 B step through the quarters by themselves.
template <int DP> __device__ __forceinline__ int xa_kx(int row) {
  return DP == 64 ? (row >> 1) & 7 : DP % 128 == 0 ? row & 7 : (row >> 2) & 3;
}
template <int DP> __device__ __forceinline__ int xa_vx(int row) {
  return DP == 64 ? ((row >> 1) & 1) << 2 : DP % 128 == 0 ? (row & 3) << 2 : 0;
}

constexpr float XA_RAISE = 8.0f;  // the running maximum is raised once a score passes it by 2^8 (p <= 256 keeps its precision in 16 bits)
// The exponent is one fma, s c - fl(m c).  The rounding of m c shifts every key's exponent alike and cancels in the quotient: by 2^-8
// at most up to |m c| = 2^16.  Past it the shift would leave p's range (it reaches 16 at 2^28; from 2^29 a row was inf over inf or 0 over
// 0), so there it is taken back, exponent by exponent: where distinct scores lie close enough to count (|m c| < 2^30) both terms are
// small and the difference is off by 2^-18 at most.  Decided for the whole wave, when a maximum is raised: 2304 rows
// to 9216 keys 110 us with it and without, heads of 32 to 333 keys 7.7 -> 7.9 ((s - m) c in a branch of its own: 112 and 8.4).
constexpr float XA_ONE_FMA = 65536.0f;

enum { XA_FULL = 0, XA_TAIL = 1, XA_REGIONS = 2 };

constexpr int XA_KT = 64;  // keys of a tile

// A SIMD's waves are in different phases: one whose matrix instructions are ready goes before one that exponentiates, or the two kinds
// wait for each other.  Heads up to 96 wide (two vector instructions' time to a matrix one's): P V first of all, 2304 rows to 9216
// keys 152 -> 137 us, heads of 80 to 4096 keys 86 -> 76.  128 and 160: Q K^T first, 126 -> 125 and 146 -> 131 (P V first: 132 and 140).
// 256: a SIMD has one wave (with any of them 156 -> 158).
enum { XA_SCORES, XA_SOFTMAX, XA_OUTPUT };
template <int DP, int PHASE> __device__ __forceinline__ void xa_priority() {
  if constexpr (DP <= 160) __builtin_amdgcn_s_setprio(PHASE == XA_SCORES ? 2 : PHASE == XA_SOFTMAX ? 0 : DP <= 96 ? 3 : 1);
}

// One wave's share of a key tile: KS blocks of 32 keys (from row kr0 of the tile) against its 32 rows.
template <int DP, int KS, int MODE>
__device__ __forceinline__ void xa_step(const u16* sK, const u16* sV, const unsigned* sR, const hx8 (&qf)[DP / 16], f32x16 (&oacc)[DP / 32], float& m,
                                        float& mc, bool& far, float& l, float c, float raise, int kr0, int key0, int klim, unsigned qset, int lane) {
  const int r = lane & 31, hh = lane >> 5, dblk = (lane >> 4) & 1, tq = (lane & 15) >> 2, tp = lane & 3;
#pragma unroll
  for (int b = 0; b < KS; ++b) {
    if (MODE != XA_FULL && KS > 1 && key0 + 32 * b >= klim) continue;  // nothing of this block is left (the same for the whole wave)
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    const int krow = kr0 + 32 * b + r;
    xa_priority<DP, XA_SCORES>();
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = MFMA32(*(const hx8*)&sK[krow * DP + (((2 * ks + hh) ^ xa_kx<DP>(krow)) << 3)], qf[ks], s, 0, 0, 0);
    xa_priority<DP, XA_SOFTMAX>();
    if constexpr (MODE == XA_TAIL) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 32 * b + 8 * (i >> 2) + 4 * hh + (i & 3) >= klim) s[i] = -__builtin_inff();
    }
    if constexpr (MODE == XA_REGIONS) {  // keys past the end carry the empty set
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x4 kr = *(const u32x4*)&sR[kr0 + 32 * b + 8 * g + 4 * hh];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(kr[e] & qset)) s[4 * g + e] = -__builtin_inff();
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    // both halves of the wave raise together: the exchange and the rescaling happen in this rare branch only
    if (__builtin_amdgcn_ballot_w64(mx - m > raise) != 0) {
      const float mnew = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
      const float alpha = __builtin_amdgcn_exp2f((m - mnew) * c);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[dt][i] *= alpha;
      m = mnew;
      mc = m == XA_LOWEST ? 0.f : m * c;  // a row that has seen nothing has scores of -inf only
      far = __builtin_amdgcn_ballot_w64(fabsf(mc) > XA_ONE_FMA) != 0;
    }
    float rs = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], c, -mc);
    if (far) {
      const float off = m == XA_LOWEST ? 0.f : __builtin_fmaf(m, c, -mc);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] -= off;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i]);
      rs += s[i];
    }
    l += rs;
    xa_priority<DP, XA_OUTPUT>();
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      hx8 pb;
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[j] = (h16)s[8 * s2 + j];
      const int vrow = kr0 + 32 * b + 16 * s2 + 4 * hh + tq;  // and vrow + 8, whose swizzle is the same
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const u16* vp = sV + vrow * DP + (((4 * dt + 2 * dblk + (tp >> 1)) ^ xa_vx<DP>(vrow)) << 3) + 4 * (tp & 1);
        union { struct { short4_t a, b; } h; hx8 v; } u;
        u.h.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)vp);
        u.h.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)(vp + 8 * DP));
        oacc[dt] = MFMA32(u.v, pb, oacc[dt], 0, 0, 0);
      }
    }
  }
}

// Block: 4 waves = 4 / WK groups of 32 rows by WK shares of every tile; the shares' (m, l, O) merge in the LDS.
template <int DP, int WK, bool REG>
struct XaShape {
  static constexpr int WR = 4 / WK, KS = XA_KT / 32 / WK, ROWS = WR * 32, BUF = 2 * XA_KT * DP;  // BUF: elements of K and V of a tile
  static constexpr int merge = WK == 1 ? 0 : 4 * 32 * (DP * 4 + 8);
  static constexpr int stage = 2 * (BUF * 2 + (REG ? XA_KT * 4 : 0));
  static constexpr int bytes = stage > merge ? stage : merge;
};
template <int DP, int WK, bool REG>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void xattn_kernel(const XattnParams p) {
  typedef XaShape<DP, WK, REG> S;
  constexpr int KT = XA_KT, CH = DP / 8, PT = KT * CH / 256;  // 16-byte pieces of a row; pieces of K (and of V) a thread moves per tile
  static_assert(KT * CH % 256 == 0 && S::KS >= 1, "tile / wave grid mismatch");
  extern __shared__ __attribute__((aligned(16))) u16 smem[];
  unsigned* const sreg = (unsigned*)(smem + 2 * S::BUF);
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), wr = wv / WK, wk = wv % WK, r = lane & 31, hh = lane >> 5;
  int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = bid % p.rtiles;
  bid /= p.rtiles;
  const int sp = bid % p.splits;
  bid /= p.splits;
  // the samples of one head follow each other: an XCD's run of blocks then holds long and short contexts alike (with the heads of one
  // sample together, contexts of 9216 and 4600 keys took as long as two of 9216), and samples that share a context meet in its L2
  const int bz = bid % p.batch, hk = bid / p.batch;
  const int ctx = p.index ? scalar_i32(p.index + bz) : (p.contexts == 1 ? 0 : bz);
  const bool ctx_ok = ctx >= 0 && ctx < p.contexts;
  const int len = !ctx_ok ? 0 : p.lens ? min(max(scalar_i32(p.lens + ctx), 0), p.nkv) : p.nkv;
  const int ntiles = (len + KT - 1) / KT;
  const int t0 = (int)((long long)ntiles * sp / p.splits), t1 = (int)((long long)ntiles * (sp + 1) / p.splits);
  const int cz = ctx_ok ? ctx : 0;
  const u16* kb = p.k + (long long)cz * p.sk + (long long)hk * p.dim;
  const u16* vb = p.v + (long long)cz * p.sv + (long long)hk * p.dim;
  const unsigned* krp = REG ? p.kreg + (long long)cz * p.skr : nullptr;

  // ---- staging by LDS-DMA, two buffers.  A key past the end reads as zeros (it lies past the descriptor's records, so memory is
  // not touched), a piece past the head's width too; so does V of a key in no region: p = 0 must not meet a NaN.
  unsigned koff[PT], voff[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int piece = t + 256 * i, row = piece / CH, ch = piece % CH, ck = ch ^ xa_kx<DP>(row), cv = ch ^ xa_vx<DP>(row);
    koff[i] = ck * 8 < p.dim ? 2u * ((unsigned)row * p.ldk + ck * 8) : DMA_OOB;
    voff[i] = cv * 8 < p.dim ? 2u * ((unsigned)row * p.ldv + cv * 8) : DMA_OOB;
  }
  const unsigned lds0 = lds_addr_of(smem) + wv * 1024;
  auto stage = [&](int tile, int buf) {
    const int key0 = tile * KT, left = min(len - key0, KT);
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(kb + (long long)key0 * p.ldk), 0, (unsigned)left * p.ldk * 2u, 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(vb + (long long)key0 * p.ldv), 0, (unsigned)left * p.ldv * 2u, 0x00020000);
    const unsigned dst = lds0 + buf * (S::BUF * 2);
    if constexpr (REG) {
      unsigned word[PT];
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        const int row = (t + 256 * i) / CH;
        word[i] = row < left ? krp[key0 + row] : 0u;
      }
      if (t < KT) sreg[buf * KT + t] = t < left ? krp[key0 + t] : 0u;
#pragma unroll
      for (int i = 0; i < PT; ++i) dma_buf16(rk, koff[i], 0, dst + i * 4096);
#pragma unroll
      for (int i = 0; i < PT; ++i) dma_buf16(rv, word[i] ? voff[i] : DMA_OOB, 0, dst + KT * DP * 2 + i * 4096);
    } else {
#pragma unroll
      for (int i = 0; i < PT; ++i) dma_buf16(rk, koff[i], 0, dst + i * 4096);
#pragma unroll
      for (int i = 0; i < PT; ++i) dma_buf16(rv, voff[i], 0, dst + KT * DP * 2 + i * 4096);
    }
  };
  // every DMA of this wave has landed and its reads of the buffer that is staged next have returned; then meet the others
#define XA_LANDED() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory")
  if (t0 < t1) stage(t0, 0);

  // ---- this wave's rows: row rho of the kv head is query rho / group, head rho % group of the group
  const int rho = rt * S::ROWS + wr * 32 + r, rc = min(rho, p.rows - 1);
  const int qi = rc / p.group, head = hk * p.group + rc % p.group;
  const u16* Q = p.q + (long long)bz * p.sq + (long long)qi * p.ldq + head * p.dim;
  hx8 qf[DP / 16];
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int d = 16 * ks + 8 * hh;
#pragma unroll
    for (int e = 0; e < 8; ++e) qf[ks][e] = (h16)0.f;
    if (d < p.dim) qf[ks] = *(const hx8*)(Q + d);
  }
  const unsigned qset = REG ? p.qreg[(long long)bz * p.sqr + qi] : 0u;
  f32x16 oacc[DP / 32];
  float m = XA_LOWEST, mc = 0.f, l = 0.f;
  bool far = false;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
  // a wave without rows only helps to move the tiles (4 x 8 heads of 256, 4 rows to 2048 keys: 24.5 -> 22.6 us)
  const bool live = rt * S::ROWS + wr * 32 < p.rows;
  const int kr0 = wk * (KT / WK), tfull = min(t1, len / KT);  // tiles below tfull are whole
  // the rows' own loads are waited for here, where the compiler sees it: it would else wait inside the loop for everything in
  // flight, the next tile's DMA among it
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  XA_LANDED();
#pragma unroll 1
  for (int tile = t0; tile < (REG ? t1 : tfull); ++tile) {
    const int cur = (tile - t0) & 1;
    if (tile + 1 < t1) stage(tile + 1, cur ^ 1);
    const u16* sK = smem + cur * S::BUF;
    if (live) xa_step<DP, S::KS, REG ? XA_REGIONS : XA_FULL>(sK, sK + KT * DP, sreg + cur * KT, qf, oacc, m, mc, far, l, p.c, p.raise, kr0, tile * KT + kr0, len, qset, lane);
    XA_LANDED();
  }
  if (!REG && live && t0 < t1 && tfull < t1) {  // the one partial tile: its data has landed
    const u16* sK = smem + ((t1 - 1 - t0) & 1) * S::BUF;
    xa_step<DP, S::KS, XA_TAIL>(sK, sK + KT * DP, sreg, qf, oacc, m, mc, far, l, p.c, p.raise, kr0, (t1 - 1) * KT + kr0, len, qset, lane);
  }
#undef XA_LANDED
  l += __shfl_xor(l, 32);

  float* const mo = (float*)smem;  // WK > 1: [wave][dt][16][64]
  if constexpr (WK > 1) {
    // merge: m and l of the rows, then each share's O scaled to the common maximum; share wk of a row group finishes the groups
    // g = wk, wk + WK, ... of every 32 columns, summing in the order of the shares
    float2* const mml = (float2*)(mo + 4 * 32 * DP);  // [wave][32]
    __syncthreads();
    if (hh == 0) mml[wv * 32 + r] = make_float2(m, l);
    __syncthreads();
    float mall = XA_LOWEST, lall = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) mall = fmaxf(mall, mml[(wr * WK + w) * 32 + r].x);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float2 v = mml[(wr * WK + w) * 32 + r];
      lall += v.y * __builtin_amdgcn_exp2f((v.x - mall) * p.c);
    }
    const float alpha = __builtin_amdgcn_exp2f((m - mall) * p.c);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mo[((wv * (DP / 32) + dt) * 16 + i) * 64 + lane] = oacc[dt][i] * alpha;
    m = mall;
    l = lall;
    __syncthreads();
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  if constexpr (WK == 1) {
    if (p.splits == 1) {
      // a lane has 8 bytes here and there of one row: turned in the wave's own piece of LDS, rows leave as whole lines (9216 rows to 77
      // keys 12.2 -> 10.9 us, 576 rows to 231 24.7 -> 22.3).  Not past the L2: 9.9 and 21.2 alone, but the projection behind them reads
      // the rows over and over (84 -> 89 us together)
      constexpr int LD = DP + 8;  // the row, then where it goes
      static_assert(4 * 32 * LD * 2 <= S::bytes, "the rows in the tiles' memory");
      u16* const so = smem + wv * 32 * LD;
      __syncthreads();
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(uint2*)&so[r * LD + 32 * dt + 8 * g + 4 * hh] = make_uint2(pack2h(oacc[dt][4 * g] * inv, oacc[dt][4 * g + 1] * inv), pack2h(oacc[dt][4 * g + 2] * inv, oacc[dt][4 * g + 3] * inv));
      if (hh == 0) *(long long*)&so[r * LD + DP] = rho < p.rows ? (long long)bz * p.so + (long long)qi * p.ldo + head * p.dim : -1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes
      typedef u32x4 u32x4_a8 __attribute__((aligned(8)));
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) {
        const int piece = 64 * i + lane, row = piece / CH, ch = piece % CH;
        const long long off = *(const long long*)&so[row * LD + DP];
        const u32x4 v = *(const u32x4*)&so[row * LD + 8 * ch];
        if (off >= 0 && 8 * ch < p.dim) *(u32x4_a8*)(p.o + off + 8 * ch) = v;
      }
      return;
    }
  }
  if (rho >= p.rows) return;
  const long long prow = ((long long)bz * p.kvh + hk) * p.rows + rho;
  float* po = p.po + (prow * p.splits + sp) * p.dim;
  u16* O = p.o + (long long)bz * p.so + (long long)qi * p.ldo + head * p.dim;
  if (p.splits > 1 && wk == 0 && hh == 0) p.pml[prow * p.splits + sp] = make_float2(m, l);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int gi = 0; gi < 4 / WK; ++gi) {
      const int g = WK * gi + wk, d = 32 * dt + 8 * g + 4 * hh;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (WK == 1) {
          y[e] = oacc[dt][4 * gi + e];
        } else {
          y[e] = 0.f;
#pragma unroll
          for (int w = 0; w < WK; ++w) y[e] += mo[(((wr * WK + w) * (DP / 32) + dt) * 16 + 4 * g + e) * 64 + lane];
        }
      }
      if (d >= p.dim) continue;
      if (p.splits > 1) *(f32x4*)(po + d) = y;
      else *(uint2*)(O + d) = make_uint2(pack2h(y[0] * inv, y[1] * inv), pack2h(y[2] * inv, y[3] * inv));
    }
}

// Joins the splits of a row, in split order: one wave per row, the splits' (m, l) on the lanes.
__global__ __launch_bounds__(256) void xattn_join_kernel(const XattnParams p, long long total) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= total) return;
  const float2 ml = lane < p.splits ? p.pml[row * p.splits + lane] : make_float2(XA_LOWEST, 0.f);
  const float mall = wave_max(ml.x);
  const float a = __builtin_amdgcn_exp2f((ml.x - mall) * p.c);
  const float l = wave_sum(a * ml.y);
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  const long long kvrow = row / p.rows;
  const int rho = (int)(row - kvrow * p.rows), hk = (int)(kvrow % p.kvh), bz = (int)(kvrow / p.kvh);
  u16* O = p.o + (long long)bz * p.so + (long long)(rho / p.group) * p.ldo + (hk * p.group + rho % p.group) * p.dim;
  const float* po = p.po + row * p.splits * p.dim;
  for (int d0 = 0; d0 < p.dim; d0 += 128) {  // every lane takes part: the weights come from all of them
    const int d = d0 + 2 * lane;
    const float* pd = po + (d < p.dim ? d : 0);
    float y0 = 0.f, y1 = 0.f;
    for (int s0 = 0; s0 < p.splits; s0 += 8) {  // eight splits' loads in flight: one memory latency for all of them
      float2 v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) v[s] = *(const float2*)(pd + (long long)min(s0 + s, p.splits - 1) * p.dim);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float as = s0 + s < p.splits ? __shfl(a, s0 + s) : 0.f;
        y0 += as * v[s].x;
        y1 += as * v[s].y;
      }
    }
    if (d < p.dim) *(uint32_t*)(O + d) = pack2h(y0 * inv, y1 * inv);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
struct XattnPlan { int wk, rtiles, splits; };
static XattnPlan xattn_plan(int batch, int kvh, int dim, int rows, int nkv) {
  XattnPlan pl;
  // one wave sweeps all keys for its 32 rows, or two waves share them.  The second gives blocks of 64 rows, fewer of them idle where
  // there are few and finer pieces where contexts differ, and pays a merge for each block.  Measured, one / two, us: heads of 64, 2304
  // rows to 154 keys 8.7 / 10.1, to 512 13.9 / 13.9, to 2304 42 / 38, to 9216 148 / 133; of 32 and of 80 to 4096 60 / 47 and 84 / 75; of 128 and of 160
  // 110 / 135 and 121 / 200; 128 heads of 64 to 512 keys, 1 row 11.7 / 10.9, 64 rows 15.6 / 15.1.  Where the rule loses: many blocks over few keys (9216
  // rows to 512 keys 21.2 / 25.1, to 1024 35.4 / 38.9), few rows to a prompt's (1 row to 77: 5.1 / 5.7, heads of 128 6.4 / 7.5), heads of 256 over 512
  // keys, which one wave cuts in two pieces (55.8 / 41.9)
  const bool few = rows <= 64;
  pl.wk = few || (dim <= 96 && nkv >= 512) ? 2 : 1;
  const int per = pl.wk == 2 ? 64 : 128;
  pl.rtiles = (rows + per - 1) / per;
  const long long blocks = (long long)batch * kvh * pl.rtiles;
  // few blocks over long states: cut the keys until the chip is full (512 blocks: two per CU), at least 256 keys to a piece.  With
  // few rows the join is cheap and the quotient is rounded up (320 blocks of one row to 9216 keys: 161 us whole, 138 + 5 in pieces)
  long long s = (few ? 511 + blocks : 512) / (blocks > 0 ? blocks : 1);
  if (s > nkv / 256) s = nkv / 256;
  if (s > 64) s = 64;
  pl.splits = s < 2 ? 1 : (int)s;
  return pl;
}

template <int DP, int WK, bool REG>
static int xattn_launch2(const XattnParams& p, int blocks, hipStream_t st) {
  constexpr int bytes = XaShape<DP, WK, REG>::bytes;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  if constexpr (bytes > 64 * 1024) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    (void)hipGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      const hipError_t e = hipFuncSetAttribute((const void*)xattn_kernel<DP, WK, REG>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != hipSuccess) {
        sdmi_set_error("cross_attention: %d bytes of LDS refused: %s", bytes, hipGetErrorString(e));
        return SDMI_ELAUNCH;
      }
      done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  hipLaunchKernelGGL((xattn_kernel<DP, WK, REG>), dim3(blocks), dim3(256), bytes, st, p);
  sdmi_note_kernel("xattn_kernel<%d, %d, %s>%s", DP, WK, REG ? "true" : "false", p.splits > 1 ? " + xattn_join_kernel" : "");
  return sdmi_check_launch("cross_attention");
}
template <int DP>
static int xattn_launch(const XattnParams& p, int wk, int blocks, hipStream_t st) {
  if (wk == 2) return p.qreg ? xattn_launch2<DP, 2, true>(p, blocks, st) : xattn_launch2<DP, 2, false>(p, blocks, st);
  return p.qreg ? xattn_launch2<DP, 1, true>(p, blocks, st) : xattn_launch2<DP, 1, false>(p, blocks, st);
}

static bool xattn_shape_ok(int batch, int heads, int kv_heads, int dim, int nq, int nkv) {
  return batch > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && dim >= 8 && dim <= 256 && dim % 8 == 0 && nq > 0 && nkv >= 0 &&
         nkv < (1 << 30) && (long long)nq * (heads / kv_heads) < (1ll << 30) && (long long)heads * dim < (1ll << 22);
}
// a launch has fewer than 2^32 threads, and products with these two stay within 64 bits
static bool xattn_grid_ok(int batch, int kv_heads) { return (long long)batch * kv_heads < (1ll << 24); }

extern "C" int64_t sdmi_cross_attention_ws_bytes(int batch, int heads, int kv_heads, int dim, int nq, int nkv) {
  if (!xattn_shape_ok(batch, heads, kv_heads, dim, nq, nkv) || !xattn_grid_ok(batch, kv_heads)) return 0;
  const XattnPlan pl = xattn_plan(batch, kv_heads, dim, nq * (heads / kv_heads), nkv);
  return pl.splits == 1 ? 0 : (int64_t)batch * heads * nq * pl.splits * ((int64_t)dim * 4 + 8);
}

extern "C" int sdmi_cross_attention(const void* q, int ldq, int64_t sq, const void* k, int ldk, int64_t sk, const void* v, int ldv, int64_t sv,
                                    void* o, int ldo, int64_t so, int batch, int contexts, int heads, int kv_heads, int dim, int nq, int nkv,
                                    const int32_t* index, const int32_t* lens, const uint32_t* query_regions, int64_t sqr,
                                    const uint32_t* key_regions, int64_t skr, float scale, void* ws, int64_t ws_bytes, void* stream) {
  SDMI_REQUIRE(q && o && (nkv == 0 || (k && v)), "cross_attention: null pointer");
  SDMI_REQUIRE(xattn_shape_ok(batch, heads, kv_heads, dim, nq, nkv),
               "cross_attention: bad shape (batch %d, %d heads on %d key heads, head width %d: a multiple of 8 up to 256, %d queries, %d keys)", batch, heads,
               kv_heads, dim, nq, nkv);
  SDMI_REQUIRE(xattn_grid_ok(batch, kv_heads), "cross_attention: grid too large");
  SDMI_REQUIRE(contexts > 0, "cross_attention: %d contexts", contexts);
  SDMI_REQUIRE(index || contexts == 1 || contexts == batch, "cross_attention: %d contexts for a batch of %d need an index", contexts, batch);
  SDMI_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 4 == 0, "cross_attention: row strides must be multiples of 8");
  SDMI_REQUIRE(ldq >= heads * dim && ldo >= heads * dim && ldk >= kv_heads * dim && ldv >= kv_heads * dim, "cross_attention: row stride < heads * dim");
  SDMI_REQUIRE(ldk < (1 << 22) && ldv < (1 << 22), "cross_attention: k/v row stride too large");  // 32-bit byte offsets inside a tile
  SDMI_REQUIRE(sq % 8 == 0 && sk % 8 == 0 && sv % 8 == 0 && so % 4 == 0, "cross_attention: batch strides must keep alignment");
  SDMI_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((uintptr_t)o & 7) == 0, "cross_attention: pointer alignment");
  SDMI_REQUIRE(!query_regions == !key_regions, "cross_attention: regions of queries and of keys go together");
  SDMI_REQUIRE((((uintptr_t)index | (uintptr_t)lens | (uintptr_t)query_regions | (uintptr_t)key_regions) & 3) == 0, "cross_attention: pointer alignment");
  // past it a softmax is a maximum; scale * log2(e) stays finite
  SDMI_REQUIRE(scale > 0.f && scale <= 1e15f, "cross_attention: scale must be positive and at most 1e15");
  XattnParams p = {};
  p.q = (const u16*)q; p.k = (const u16*)k; p.v = (const u16*)v; p.o = (u16*)o;
  p.sq = sq; p.sk = sk; p.sv = sv; p.so = so; p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
  p.batch = batch; p.contexts = contexts; p.heads = heads; p.kvh = kv_heads; p.group = heads / kv_heads; p.dim = dim; p.nq = nq; p.nkv = nkv;
  p.rows = nq * p.group;
  p.index = index; p.lens = lens; p.qreg = query_regions; p.kreg = key_regions; p.sqr = sqr; p.skr = skr;
  p.c = scale * 1.44269504088896340736f;
  p.raise = fminf(XA_RAISE / p.c, XA_RAISE_MAX);
  XattnPlan pl = xattn_plan(batch, kv_heads, dim, p.rows, nkv);
  const int64_t prows = (int64_t)batch * heads * nq;
  if (pl.splits > 1 && (!ws || ws_bytes < prows * pl.splits * ((int64_t)dim * 4 + 8))) pl.splits = 1;  // as with split-K: no room, no split
  SDMI_REQUIRE(pl.splits == 1 || ((uintptr_t)ws & 15) == 0, "cross_attention: workspace alignment");
  p.rtiles = pl.rtiles; p.splits = pl.splits;
  p.po = (float*)ws;
  p.pml = pl.splits > 1 ? (float2*)((float*)ws + prows * pl.splits * dim) : nullptr;
  const long long blocks = (long long)batch * kv_heads * pl.rtiles * pl.splits;
  SDMI_REQUIRE(blocks < (1ll << 24) && (pl.splits == 1 || (prows + 3) / 4 < (1ll << 24)), "cross_attention: grid too large");
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (dim <= 32) rc = xattn_launch<32>(p, pl.wk, (int)blocks, st);
  else if (dim <= 64) rc = xattn_launch<64>(p, pl.wk, (int)blocks, st);
  else if (dim <= 96) rc = xattn_launch<96>(p, pl.wk, (int)blocks, st);
  else if (dim <= 128) rc = xattn_launch<128>(p, pl.wk, (int)blocks, st);
  else if (dim <= 160) rc = xattn_launch<160>(p, pl.wk, (int)blocks, st);
  else rc = xattn_launch<256>(p, pl.wk, (int)blocks, st);
  if (rc != SDMI_OK || pl.splits == 1) return rc;
  hipLaunchKernelGGL(xattn_join_kernel, dim3((unsigned)((prows + 3) / 4)), dim3(256), 0, st, p, (long long)prows);
  return sdmi_check_launch("cross_attention (join)");
}

extern "C" int sdmi_cross_attention_packed(const sdmi_cross_attention_args* a) {
  SDMI_REQUIRE(a, "cross_attention: null pointer");
  SDMI_REQUIRE(sdmi_fits_int(a->ldq) && sdmi_fits_int(a->ldk) && sdmi_fits_int(a->ldv) && sdmi_fits_int(a->ldo) && sdmi_fits_int(a->batch) && sdmi_fits_int(a->contexts) &&
                   sdmi_fits_int(a->heads) && sdmi_fits_int(a->kv_heads) && sdmi_fits_int(a->dim) && sdmi_fits_int(a->nq) && sdmi_fits_int(a->nkv),
               "cross_attention: bad shape (a size or row stride past 32 bits)");
  return sdmi_cross_attention(a->q, (int)a->ldq, a->sq, a->k, (int)a->ldk, a->sk, a->v, (int)a->ldv, a->sv, a->o, (int)a->ldo, a->so, (int)a->batch, (int)a->contexts,
                              (int)a->heads, (int)a->kv_heads, (int)a->dim, (int)a->nq, (int)a->nkv, a->index, a->lens, a->query_regions, a->sqr, a->key_regions, a->skr,
                              (float)a->scale, a->ws, a->ws_bytes, a->stream);
}
