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
// Mathematics: one pass over the keys with the running maximum m and sum l of the softmax, in base 2 (scale * log2(e) enters
// the exponent's fma in fp32; q and k are multiplied as they are).  S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: the
// query is on the lane in both, so the statistics are lane-local plus one exchange of the wave's halves, and P leaves the
// first product in the operand layout of the second (k order inside a 16-key step as the accumulator has it; V is read
// through ds_read_b64_tr_b16 in that order).  P is rounded to 16 bits for the matrix cores (half a step of a value <= 1);
// S, m, l and O stay in fp32.
#include "common.h"
#include <atomic>

struct XattnParams {
  const u16 *q, *k, *v;
  u16* o;
  long long sq, sk, sv, so;
  int ldq, ldk, ldv, ldo;
  int contexts, heads, kvh, group, dim, nq, nkv, rows, rtiles, splits;  // rows = nq * group: the rows of one kv head
  const int *index, *lens;
  const unsigned *qreg, *kreg;
  long long sqr, skr;
  float c;  // scale * log2(e)
  float* po;    // splits > 1: [row][split][dim] un-normalised partial outputs
  float2* pml;  // [row][split] (m, l)
};

constexpr float XA_LOWEST = -1e30f;  // start of the running maximum: below every scaled score, and finite, so that m - m is 0

// LDS row strides in elements.  K: fragment reads are 16 B at the same column of 8 consecutive rows: (DP + 8) / 2 dwords is
// 4 mod 8, which spreads them over the banks.  V: a transposed read takes 4 rows x 64 B: stride 16 or 48 dwords mod 64.
template <int DP> constexpr int xa_kstr() { return DP + 8; }
template <int DP> constexpr int xa_vstr() { return (DP / 2) % 64 == 16 || (DP / 2) % 64 == 48 ? DP : DP + 32; }

enum { XA_FULL = 0, XA_TAIL = 1, XA_REGIONS = 2 };

// One wave's share of a key tile: KS blocks of 32 keys against its 32 rows.
template <int DP, int KS, int MODE>
__device__ __forceinline__ void xa_step(const u16* sK, const u16* sV, const unsigned* sR, const hx8 (&qf)[DP / 16], f32x16 (&oacc)[DP / 32],
                                        float& m, float& l, float c, int key0, int klim, unsigned qset, int lane) {
  constexpr int KSTR = xa_kstr<DP>(), VSTR = xa_vstr<DP>();
  const int r = lane & 31, hh = lane >> 5, dblk = (lane >> 4) & 1, tq = (lane & 15) >> 2, tp = lane & 3;
  f32x16 s[KS];
#pragma unroll
  for (int b = 0; b < KS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
    for (int b = 0; b < KS; ++b) s[b] = MFMA32(*(const hx8*)&sK[(32 * b + r) * KSTR + 16 * ks + 8 * hh], qf[ks], s[b], 0, 0, 0);
  if constexpr (MODE == XA_TAIL) {
#pragma unroll
    for (int b = 0; b < KS; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 32 * b + 8 * (i >> 2) + 4 * hh + (i & 3) >= klim) s[b][i] = -__builtin_inff();
  }
  if constexpr (MODE == XA_REGIONS) {  // keys past the end carry the empty set
#pragma unroll
    for (int b = 0; b < KS; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x4 kr = *(const u32x4*)&sR[32 * b + 8 * g + 4 * hh];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(kr[e] & qset)) s[b][4 * g + e] = -__builtin_inff();
      }
  }
  float mx = s[0][0];
#pragma unroll
  for (int b = 0; b < KS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const float mnew = fmaxf(m, mx * c);
  // no lane's maximum moved (the usual case after a few tiles): nothing to rescale
  if (__builtin_amdgcn_ballot_w64(mnew > m) != 0) {
    const float alpha = __builtin_amdgcn_exp2f(m - mnew);
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[dt][i] *= alpha;
    m = mnew;
  }
  float rs = 0.f;
#pragma unroll
  for (int b = 0; b < KS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], c, -m));
      s[b][i] = e;
      rs += e;
    }
  l += rs;
#pragma unroll
  for (int b = 0; b < KS; ++b)
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      hx8 pb;
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[j] = (h16)s[b][8 * s2 + j];
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const u16* vp = sV + (32 * b + 16 * s2 + 4 * hh + tq) * VSTR + 32 * dt + 16 * dblk + 4 * tp;
        union { struct { short4_t a, b; } h; hx8 v; } u;
        u.h.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)vp);
        u.h.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((short4_t __attribute__((address_space(3)))*)(vp + 8 * VSTR));
        oacc[dt] = MFMA32(u.v, pb, oacc[dt], 0, 0, 0);
      }
    }
}

template <int DP, int WK> constexpr int xa_tile_keys() { return WK == 1 ? 64 : 128; }
template <int DP, int WK> constexpr int xa_bufs() { return xa_tile_keys<DP, WK>() * (xa_kstr<DP>() + xa_vstr<DP>()) * 2 * 2 <= 80 * 1024 ? 2 : 1; }
template <int DP, int WK> constexpr int xa_lds_bytes() {
  constexpr int stage = xa_bufs<DP, WK>() * xa_tile_keys<DP, WK>() * ((xa_kstr<DP>() + xa_vstr<DP>()) * 2 + 4);
  constexpr int merge = WK == 1 ? 0 : 4 * 32 * DP * 4 + 4 * 32 * 8;
  return stage > merge ? stage : merge;
}

// Block: 4 waves.  WK = 1: each wave owns 32 of the block's 128 rows and sweeps all keys.  WK = 4: the block has 32 rows, each
// wave sweeps a quarter of every key tile (few rows, long states: one query, decoding), the waves' (m, l, O) merge in the LDS.
template <int DP, int WK, bool REG>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void xattn_kernel(const XattnParams p) {
  constexpr int KT = xa_tile_keys<DP, WK>(), KS = KT / 32 / WK, KSTR = xa_kstr<DP>(), VSTR = xa_vstr<DP>(), NB = xa_bufs<DP, WK>();
  constexpr int CH = DP / 8, PT = KT * CH / 256;  // 16-byte pieces of a row; pieces of K (and of V) a thread stages per tile
  constexpr int BUF = KT * (KSTR + VSTR);         // elements per buffer
  extern __shared__ __attribute__((aligned(16))) u16 smem[];
  unsigned* const sreg = (unsigned*)(smem + NB * BUF);
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, r = lane & 31, hh = lane >> 5;
  int bid = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = bid % p.rtiles;
  bid /= p.rtiles;
  const int sp = bid % p.splits;
  bid /= p.splits;
  const int hk = bid % p.kvh, bz = bid / p.kvh;
  const int ctx = p.index ? p.index[bz] : (p.contexts == 1 ? 0 : bz);
  const bool ctx_ok = ctx >= 0 && ctx < p.contexts;
  const int len = !ctx_ok ? 0 : p.lens ? min(max(p.lens[ctx], 0), p.nkv) : p.nkv;
  const int ntiles = (len + KT - 1) / KT;
  const int t0 = (int)((long long)ntiles * sp / p.splits), t1 = (int)((long long)ntiles * (sp + 1) / p.splits);
  const int cz = ctx_ok ? ctx : 0;
  const char* kb = (const char*)(p.k + (long long)cz * p.sk + (long long)hk * p.dim);
  const char* vb = (const char*)(p.v + (long long)cz * p.sv + (long long)hk * p.dim);
  const unsigned* krp = REG ? p.kreg + (long long)cz * p.skr : nullptr;

  // ---- this wave's rows: row rho of the kv head is query rho / group, head rho % group of the group
  const int rho = (rt * (WK == 1 ? 4 : 1) + (WK == 1 ? wv : 0)) * 32 + r;
  const bool row_ok = rho < p.rows;
  const int qi = (row_ok ? rho : p.rows - 1) / p.group, head = hk * p.group + (row_ok ? rho : p.rows - 1) % p.group;
  const u16* Q = p.q + (long long)bz * p.sq + (long long)qi * p.ldq + head * p.dim;
  hx8 qf[DP / 16];
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int d = 16 * ks + 8 * hh;
#pragma unroll
    for (int e = 0; e < 8; ++e) qf[ks][e] = (h16)0.f;
    if (d < p.dim) qf[ks] = *(const hx8*)(Q + d);
  }
  const unsigned qset = REG ? (row_ok ? p.qreg[(long long)bz * p.sqr + qi] : 0u) : 0u;

  // ---- staging through registers: the next tile's loads are in flight under this tile's products.  A key past the end (or
  // in no region) is staged as zeros whatever memory holds there: p = 0 must not meet a NaN in the second product.
  unsigned koff[PT], voff[PT];
  int srow[PT];
  bool cok[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int piece = t + 256 * i, row = piece / CH, ch = piece % CH;
    srow[i] = row;
    cok[i] = ch * 8 < p.dim;
    koff[i] = 2u * ((unsigned)row * p.ldk + ch * 8);
    voff[i] = 2u * ((unsigned)row * p.ldv + ch * 8);
  }
  u32x4 kreg_[PT], vreg_[PT];
  unsigned rreg = 0;
  auto load = [&](int tile) {
    const int key0 = tile * KT;
    const char* kt = kb + (long long)key0 * p.ldk * 2;
    const char* vt = vb + (long long)key0 * p.ldv * 2;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      kreg_[i] = vreg_[i] = u32x4{0u, 0u, 0u, 0u};
      if (key0 + srow[i] < len && cok[i]) {
        kreg_[i] = *(const u32x4*)(kt + koff[i]);
        vreg_[i] = *(const u32x4*)(vt + voff[i]);
        if (REG && krp[key0 + srow[i]] == 0) kreg_[i] = vreg_[i] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    if (REG && t < KT) rreg = key0 + t < len ? krp[key0 + t] : 0u;
  };
  auto store = [&](int buf) {
    u16* sK = smem + buf * BUF;
    u16* sV = sK + KT * KSTR;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int piece = t + 256 * i, row = piece / CH, ch = piece % CH;
      *(u32x4*)&sK[row * KSTR + ch * 8] = kreg_[i];
      *(u32x4*)&sV[row * VSTR + ch * 8] = vreg_[i];
    }
    if (REG && t < KT) sreg[buf * KT + t] = rreg;
  };

  f32x16 oacc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;
  float m = XA_LOWEST, l = 0.f;
  if (t0 < t1) {
    load(t0);
    store(0);
  }
  __syncthreads();
  for (int tile = t0; tile < t1; ++tile) {
    const int cur = NB == 2 ? (tile - t0) & 1 : 0;
    if (tile + 1 < t1) load(tile + 1);
    const u16* sK = smem + cur * BUF + (WK == 1 ? 0 : wv * 32 * KSTR);
    const u16* sV = smem + cur * BUF + KT * KSTR + (WK == 1 ? 0 : wv * 32 * VSTR);
    const int key0 = tile * KT + (WK == 1 ? 0 : wv * 32);
    if constexpr (REG) {
      xa_step<DP, KS, XA_REGIONS>(sK, sV, sreg + cur * KT + (WK == 1 ? 0 : wv * 32), qf, oacc, m, l, p.c, key0, len, qset, lane);
    } else {
      if (tile * KT + KT <= len) xa_step<DP, KS, XA_FULL>(sK, sV, nullptr, qf, oacc, m, l, p.c, key0, len, 0u, lane);
      else xa_step<DP, KS, XA_TAIL>(sK, sV, nullptr, qf, oacc, m, l, p.c, key0, len, 0u, lane);
    }
    if (tile + 1 < t1) {
      if constexpr (NB == 1) __syncthreads();
      store(NB == 2 ? cur ^ 1 : 0);
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 32);
  const long long prow = ((long long)bz * p.kvh + hk) * p.rows + rho;
  u16* O = p.o + (long long)bz * p.so + (long long)qi * p.ldo + head * p.dim;

  if constexpr (WK == 1) {
    if (!row_ok) return;
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    if (p.splits > 1) {
      if (hh == 0) p.pml[prow * p.splits + sp] = make_float2(m, l);
      float* po = p.po + (prow * p.splits + sp) * p.dim;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * dt + 8 * g + 4 * hh;
          if (d < p.dim) *(f32x4*)(po + d) = f32x4{oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]};
        }
      return;
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * dt + 8 * g + 4 * hh;
        if (d < p.dim)
          *(uint2*)(O + d) = make_uint2(pack2h(oacc[dt][4 * g] * inv, oacc[dt][4 * g + 1] * inv), pack2h(oacc[dt][4 * g + 2] * inv, oacc[dt][4 * g + 3] * inv));
      }
  } else {
    // merge the four waves: m and l of the 32 rows, then each wave's O scaled to the common maximum, summed in wave order
    float* const mo = (float*)smem;                    // [wave][dt][16][64]
    float2* const mml = (float2*)(mo + 4 * 32 * DP);   // [wave][32]
    __syncthreads();
    if (hh == 0) mml[wv * 32 + r] = make_float2(m, l);
    __syncthreads();
    float2 w4[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) w4[w] = mml[w * 32 + r];
    const float mall = fmaxf(fmaxf(w4[0].x, w4[1].x), fmaxf(w4[2].x, w4[3].x));
    float lall = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) lall += w4[w].y * __builtin_amdgcn_exp2f(w4[w].x - mall);
    const float alpha = __builtin_amdgcn_exp2f(m - mall);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mo[((wv * (DP / 32) + dt) * 16 + i) * 64 + lane] = oacc[dt][i] * alpha;
    __syncthreads();
    if (!row_ok) return;
    const float inv = lall > 0.f ? 1.0f / lall : 0.f;
    if (p.splits > 1 && wv == 0 && hh == 0) p.pml[prow * p.splits + sp] = make_float2(mall, lall);
    float* po = p.po + (prow * p.splits + sp) * p.dim;
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {  // wave w finishes the groups g = w of every 32 columns
      const int d = 32 * x + 8 * wv + 4 * hh;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) y[e] += mo[((w * (DP / 32) + x) * 16 + 4 * wv + e) * 64 + lane];
      }
      if (d < p.dim) {
        if (p.splits > 1) *(f32x4*)(po + d) = f32x4{y[0], y[1], y[2], y[3]};
        else *(uint2*)(O + d) = make_uint2(pack2h(y[0] * inv, y[1] * inv), pack2h(y[2] * inv, y[3] * inv));
      }
    }
  }
}

// Joins the splits of a row, in split order: one wave per row, the splits' (m, l) on the lanes.
__global__ __launch_bounds__(256) void xattn_join_kernel(const XattnParams p, long long total) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= total) return;
  const float2 ml = lane < p.splits ? p.pml[row * p.splits + lane] : make_float2(XA_LOWEST, 0.f);
  const float mall = wave_max(ml.x);
  const float a = __builtin_amdgcn_exp2f(ml.x - mall);
  const float l = wave_sum(a * ml.y);
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  const long long kvrow = row / p.rows;
  const int rho = (int)(row - kvrow * p.rows), hk = (int)(kvrow % p.kvh), bz = (int)(kvrow / p.kvh);
  u16* O = p.o + (long long)bz * p.so + (long long)(rho / p.group) * p.ldo + (hk * p.group + rho % p.group) * p.dim;
  const float* po = p.po + row * p.splits * p.dim;
  for (int d0 = 0; d0 < p.dim; d0 += 128) {  // every lane takes part: the weights come from all of them
    const int d = d0 + 2 * lane;
    float y0 = 0.f, y1 = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      const float as = __shfl(a, s);
      const float2 v = d < p.dim ? *(const float2*)(po + (long long)s * p.dim + d) : make_float2(0.f, 0.f);
      y0 += as * v.x;
      y1 += as * v.y;
    }
    if (d < p.dim) *(uint32_t*)(O + d) = pack2h(y0 * inv, y1 * inv);
  }
}

// ------------------------------------------------------------------------------------------------------------ host
struct XattnPlan { int wk, rtiles, splits; };
static XattnPlan xattn_plan(int batch, int kvh, int rows, int nkv) {
  XattnPlan pl;
  pl.wk = rows <= 64 ? 4 : 1;
  pl.rtiles = (rows + (pl.wk == 4 ? 31 : 127)) / (pl.wk == 4 ? 32 : 128);
  const long long blocks = (long long)batch * kvh * pl.rtiles;
  // few rows over long states: cut the keys until the chip is full (512 blocks: two per CU), at least 256 keys to a piece
  long long s = 512 / (blocks > 0 ? blocks : 1);
  if (s > nkv / 256) s = nkv / 256;
  if (s > 64) s = 64;
  pl.splits = s < 2 ? 1 : (int)s;
  return pl;
}

template <int DP, int WK, bool REG>
static int xattn_launch2(const XattnParams& p, int blocks, hipStream_t st) {
  constexpr int bytes = xa_lds_bytes<DP, WK>();
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
  if (wk == 4) return p.qreg ? xattn_launch2<DP, 4, true>(p, blocks, st) : xattn_launch2<DP, 4, false>(p, blocks, st);
  return p.qreg ? xattn_launch2<DP, 1, true>(p, blocks, st) : xattn_launch2<DP, 1, false>(p, blocks, st);
}

static bool xattn_shape_ok(int batch, int heads, int kv_heads, int dim, int nq, int nkv) {
  return batch > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && dim >= 8 && dim <= 256 && dim % 8 == 0 && nq > 0 && nkv >= 0 &&
         (long long)nq * (heads / kv_heads) < (1ll << 30) && (long long)heads * dim < (1ll << 22);
}

extern "C" int64_t sdmi_cross_attention_ws_bytes(int batch, int heads, int kv_heads, int dim, int nq, int nkv) {
  if (!xattn_shape_ok(batch, heads, kv_heads, dim, nq, nkv)) return 0;
  const XattnPlan pl = xattn_plan(batch, kv_heads, nq * (heads / kv_heads), nkv);
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
  SDMI_REQUIRE(contexts > 0, "cross_attention: %d contexts", contexts);
  SDMI_REQUIRE(index || contexts == 1 || contexts == batch, "cross_attention: %d contexts for a batch of %d need an index", contexts, batch);
  SDMI_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 4 == 0, "cross_attention: row strides must be multiples of 8");
  SDMI_REQUIRE(ldq >= heads * dim && ldo >= heads * dim && ldk >= kv_heads * dim && ldv >= kv_heads * dim, "cross_attention: row stride < heads * dim");
  SDMI_REQUIRE(ldk < (1 << 22) && ldv < (1 << 22), "cross_attention: k/v row stride too large");  // 32-bit byte offsets inside a tile
  SDMI_REQUIRE(sq % 8 == 0 && sk % 8 == 0 && sv % 8 == 0 && so % 4 == 0, "cross_attention: batch strides must keep alignment");
  SDMI_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((uintptr_t)o & 7) == 0, "cross_attention: pointer alignment");
  SDMI_REQUIRE(!query_regions == !key_regions, "cross_attention: regions of queries and of keys go together");
  SDMI_REQUIRE((((uintptr_t)index | (uintptr_t)lens | (uintptr_t)query_regions | (uintptr_t)key_regions) & 3) == 0, "cross_attention: pointer alignment");
  SDMI_REQUIRE(scale > 0.f && scale < 1e30f, "cross_attention: scale must be positive and finite");
  XattnParams p = {};
  p.q = (const u16*)q; p.k = (const u16*)k; p.v = (const u16*)v; p.o = (u16*)o;
  p.sq = sq; p.sk = sk; p.sv = sv; p.so = so; p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
  p.contexts = contexts; p.heads = heads; p.kvh = kv_heads; p.group = heads / kv_heads; p.dim = dim; p.nq = nq; p.nkv = nkv;
  p.rows = nq * p.group;
  p.index = index; p.lens = lens; p.qreg = query_regions; p.kreg = key_regions; p.sqr = sqr; p.skr = skr;
  p.c = scale * 1.44269504088896340736f;
  XattnPlan pl = xattn_plan(batch, kv_heads, p.rows, nkv);
  const int64_t prows = (int64_t)batch * heads * nq;
  if (pl.splits > 1 && (!ws || ws_bytes < prows * pl.splits * ((int64_t)dim * 4 + 8))) pl.splits = 1;  // as with split-K: no room, no split
  SDMI_REQUIRE(pl.splits == 1 || ((uintptr_t)ws & 15) == 0, "cross_attention: workspace alignment");
  p.rtiles = pl.rtiles; p.splits = pl.splits;
  p.po = (float*)ws;
  p.pml = pl.splits > 1 ? (float2*)((float*)ws + prows * pl.splits * dim) : nullptr;
  const long long blocks = (long long)batch * kv_heads * pl.rtiles * pl.splits;
  SDMI_REQUIRE(blocks < (1ll << 31) && (prows + 3) / 4 < (1ll << 31), "cross_attention: grid too large");
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
