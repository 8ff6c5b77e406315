// Attention with score rules, backward: stof_score_attn_bwd (see score_attn.h for the rule).
//
// With P = softmax, dP = dO V^T and delta_i = sum_j P_ij dP_ij (= sum_d dO_id O_id):
//     dS = P (dP - delta),   dV = P^T dO,   d table[h][x] = sum of dS over the pairs of clipped distance x,
//     dT = dS (1 - tanh^2) with a cap,   dQ = scale dT K,   dK = scale dT^T Q
// P is formed again from the scores and the forward pass's lse.  Two kernels, one that owns query rows
// (dQ, delta) and then one that owns keys (dK, dV, table): each adds its sums in a fixed order, without
// atomics, so the same inputs give the same bits; the price is that S and dP are formed twice.
//
// A wave owns 32 queries (keys) and its lane one of them, as in the forward pass: S^T = K Q^T and
// dP^T = V dO^T (S = Q K^T and dP = dO V^T) leave the accumulators in the layout that the products with
// K^T (with dO^T and Q^T) take as their B operand, their A operands come from the same LDS tiles through
// the transposing read.
//
// dT enters its products in the tensors' format.  In fp16 its small values would vanish (P of long rows is
// below 1e-4) and its large ones overflow, so it carries a power of two that is taken out of the sums
// again: |dT| <= 2 D max|dO| max|V| =: bound, with the maximum of V over all keys of the head (delta holds
// them all), and dT 2^k with k = 14 - ceil(log2 bound) stays below 2^15 and keeps 11 bits down to 2^-29 of the
// bound.  P is carried as 2^12 P.  bfloat16 needs neither.
#include "score_attn.h"

#include <type_traits>

namespace {

struct BwdParams {
  ScoreParams s;
  const half_t* dout; const half_t* o; const float* lse;
  int64_t dos[3], oos[3];
  half_t* dq; half_t* dk; half_t* dv;        // contiguous [B, Hq, Sq, D], [B, Hkv, Sk, D]
  floatx2_t* stats;                          // [B, Hq, 64 ceil(Sq / 64)]: (lse in log2 units less lse_add, delta); +inf = a row without keys or past the end
  float* vmax; float* domax;                 // fp16: largest |V| per (b, hk, key block), largest |dO| per (b, h, query block)
  float* tab_part; half_t* dtable;           // per (b, h), key tile and split: sums of the 2 R + 1 distances
  float scale;
  int q_tiles, k_tiles, q_chunk, k_chunk;
  int ranges;                                // document ranges to form (0: none)
  int splits; float* kv_part;                // workgroups that share a key tile; their fp32 sums, [2][splits][B Hkv Sk D]
};

constexpr int kPShift = 12;                  // fp16: P is carried as 2^12 P
// ceil(log2 x) for the range bounds; 0 for zero, infinite or NaN arguments (nothing to protect)
__device__ __forceinline__ int ceil_log2(float x) {
  if (!(x > 0.f) || x > 3e38f) return 0;
  return (int)((__builtin_bit_cast(unsigned, x) >> 23) & 255) - 126;
}
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
// k of the header comment, held where its reciprocal is a normal number
template <int D> __device__ __forceinline__ int dt_shift(float mdo, float mv) {
  return min(max(14 - (D == 64 ? 7 : 8) - ceil_log2(mdo) - ceil_log2(mv), -100), 100);
}

// Per row of dO: (lse in log2 units, delta), and for fp16 the largest |dO| and |V| of every 64 rows.
// Also the document ranges, one per wave.  Grid: B Hq ceil(Sq / 64) workgroups of query rows, then (fp16) B Hkv ceil(Sk / 64) of value
// rows, then a quarter of the ranges.
template <int D, bool BF>
__global__ __launch_bounds__(256) void score_attn_bwd_prep_kernel(const BwdParams p) {
  const ScoreParams& s = p.s;
  constexpr int kC = D / 8;                       // lanes per row
  constexpr int kR = 64 / kC;                     // rows per wave and pass
  __shared__ float mx_lds[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane % kC;
  const int nq = (s.Sq + 63) / 64, nk = (s.Sk + 63) / 64;
  const bool is_q = (int)blockIdx.x < s.B * s.Hq * nq;
  const int range0 = s.B * s.Hq * nq + (BF ? 0 : s.B * s.Hkv * nk);
  if ((int)blockIdx.x >= range0) {
    const int n = 4 * ((int)blockIdx.x - range0) + wave;
    if (n < p.ranges) write_doc_range(s, n, lane);
    return;
  }
  float mx = 0.f;
  if (is_q) {
    const int bh = blockIdx.x / nq, t = blockIdx.x - bh * nq;
    const int b = bh / s.Hq, h = bh - b * s.Hq;
    for (int x = 0; x < 64 / (4 * kR); ++x) {
      const int r = 64 * t + (4 * x + wave) * kR + lane / kC;
      const float l = r < s.Sq ? p.lse[(int64_t)bh * s.Sq + r] : -INFINITY;
      float d = 0.f, m = 0.f;
      if (l != -INFINITY) {
        const half8_t a = *reinterpret_cast<const half8_t*>(p.dout + b * p.dos[0] + h * p.dos[1] + (int64_t)r * p.dos[2] + 8 * c);
        const half8_t y = *reinterpret_cast<const half8_t*>(p.o + b * p.oos[0] + h * p.oos[1] + (int64_t)r * p.oos[2] + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const half_t ae = a[e], ye = y[e];
          d = __builtin_fmaf(from_elem<BF>(ae), from_elem<BF>(ye), d);
          m = fmaxf(m, __builtin_fabsf(from_elem<BF>(ae)));
        }
      }
#pragma unroll
      for (int o = 1; o < kC; o <<= 1) d += __shfl_xor(d, o, 64);
      mx = fmaxf(mx, m);
      if (c == 0) p.stats[(int64_t)bh * (64 * nq) + r] = floatx2_t{l == -INFINITY ? INFINITY : __builtin_fmaf(l, kLog2e, -s.lse_add), d};
    }
  } else {
    const int idx = blockIdx.x - s.B * s.Hq * nq, bh = idx / nk, t = idx - bh * nk;
    const int b = bh / s.Hkv, h = bh - b * s.Hkv;
    const int klen = sample_of(s, b).keys;
    for (int x = 0; x < 64 / (4 * kR); ++x) {
      const int r = 64 * t + (4 * x + wave) * kR + lane / kC;
      if (r < klen && (!s.docs_k || s.docs_k[(int64_t)b * s.Sk + r] >= 0)) {
        const half8_t a = *reinterpret_cast<const half8_t*>(s.v + b * s.vs[0] + h * s.vs[1] + (int64_t)r * s.vs[2] + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) { const half_t ae = a[e]; mx = fmaxf(mx, __builtin_fabsf(from_elem<BF>(ae))); }
      }
    }
  }
  if constexpr (!BF) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if (lane == 0) mx_lds[wave] = mx;
    __syncthreads();
    if (threadIdx.x == 0) {
      mx = fmaxf(fmaxf(mx_lds[0], mx_lds[1]), fmaxf(mx_lds[2], mx_lds[3]));
      if (is_q) p.domax[blockIdx.x] = mx;
      else p.vmax[blockIdx.x - s.B * s.Hq * nq] = mx;
    }
  }
}

// Largest of n floats, to every lane of the wave.
__device__ __forceinline__ float wave_max_of(const float* a, int n) {
  float m = 0.f;
  for (int x = threadIdx.x & 63; x < n; x += 64) m = fmaxf(m, a[x]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  return m;
}

// Caps 16 raw products and leaves 1 - tanh^2 of each in w (without a cap: nothing to do, w = 1 is not read).
__device__ __forceinline__ void cap_scores_grad(const ScoreParams& p, floatx16& s, floatx16& w) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = capped(p, s[r]);
    w[r] = -4.f * __builtin_fmaf(s[r], s[r], s[r]);
  }
}

// A step works on a tile's two pieces of 32 rows (pieces 0 and 1) in four phases of D / 16 slices with two
// MFMAs each, scores and dP or sums.  Pipelined order (head size 128 without a table):
//     0: scores and dP of piece 0      1: those of piece 1, and the softmax of piece 0
//     2: sums of piece 0, and the softmax of piece 1      3: sums of piece 1
// so that in phases 1 and 2 the vector arithmetic stands between MFMAs it does not depend on: one wave lives
// on a SIMD there (its accumulators and operands fill more than 256 registers) and nothing else would fill
// the matrix pipeline meanwhile.  Plain order (head size 64, where two waves share a SIMD and 256
// registers do not hold both pieces; and with a table): piece 0, then piece 1.  The LDS fragments of a
// slice are requested two slices ahead, in a ring of three; scheduling fences between slices keep that order.
template <bool PIPE> struct Phases {
  static __device__ __forceinline__ constexpr bool scores(int ph) { return PIPE ? ph < 2 : (ph & 1) == 0; }
  static __device__ __forceinline__ constexpr int piece(int ph) { return PIPE ? ph & 1 : ph >> 1; }
};
#define STOF_FENCE() __builtin_amdgcn_sched_barrier(0)

// fragment n = s2 * (D / 32) + dt of 32 transposed rows
template <int D> __device__ __forceinline__ half8_t frag_tr(const lds_byte* t, int n, const int (&tr)[D / 32][2]) {
  const int s2 = n / (D / 32), dt = n % (D / 32);
  return lds_frag_tr(t + 16 * s2 * (2 * D) + tr[dt][0], t + 16 * s2 * (2 * D) + tr[dt][1]);
}
__device__ __forceinline__ floatx16 zero16() {
  floatx16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
  return s;
}

// 32 gradient rows of a wave through its LDS stage (rows of 2 D bytes) to contiguous rows at dst
template <int D, bool BF>
__device__ __forceinline__ void store_rows(const floatx16 (&o)[D / 32], float mul, lds_byte* stage, half_t* dst, int rows, int lane) {
  constexpr int kC = D / 8;
  const int j32 = lane & 31, g = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      half4_t o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) o4[e] = to_elem<BF>(o[dt][4 * q4 + e] * mul);
      *reinterpret_cast<__attribute__((address_space(3))) half4_t*>(stage + j32 * (2 * D) + (((4 * dt + q4) ^ (j32 & (kC - 1))) << 4) + 8 * g) = o4;
    }
  const __amdgpu_buffer_rsrc_t rs = stof_wave_rsrc(dst);
#pragma unroll
  for (int n = 0; n < 32 * kC / 64; ++n) {
    const int t = (64 / kC) * n + lane / kC, c = lane % kC;
    const half8_t v = lds_frag(stage + t * (2 * D) + ((c ^ (t & (kC - 1))) << 4));
    if (t < rows) stof_store16_through(rs, (uint32_t)t * (2 * D) + 16 * c, v);
  }
}

// ---- queries: dQ and the exact delta.  128 queries of one head per workgroup, 32 per wave; walks the key tiles as the
// forward pass's wide form does.
//
// delta from the stored output carries the output's rounding (and that of the forward pass's P): relative to
// a row whose softmax is peaked, where dP - delta is a small difference, that is several times the rounding
// of dS itself (packed documents, bfloat16: dQ and dK 4.7e-3 off where rounding them alone is 1.7e-3).  So
// delta' = sum_j P_ij dP_ij is formed along the way in fp32, and with M = P (1 - tanh^2) K as one product more
//     dQ = scale (dT(delta) K - (delta' - delta) M)
// is exact in delta while the second term stays small.  delta' replaces delta for the kernel of the keys.
//
// Bound: MFMA and vector issue, 4 products of 2 D FLOP a pair.  bf16, B2 H16 S2048: D64 80 us (860 TFLOP/s, MFMA busy 51 %), D128
// 133 us (1030 TFLOP/s, 50 %; one workgroup of four waves per unit, whose accumulators take 380 registers).
template <int D, bool BF, bool CAP, int BIAS>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void score_attn_bwd_q_kernel(const BwdParams bp) {
  const ScoreParams& p = bp.s;
  typedef TileLoad<D, kBlock, 4> TL;
  __shared__ __attribute__((aligned(1024))) unsigned char k0[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char k1[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char v0[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char v1[TL::kBytes];
  __shared__ int doc_ids[4][kBlock];
  extern __shared__ float tab[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;
  Placed at;
  if (!place(blockIdx.x, p.B * p.Hq, p.group, bp.q_tiles, bp.q_chunk, p.cus_per_xcd, D == 64 ? 2 : 1, p.causal, p.uneven, at)) return;
  const int bh = at.head, tile = bp.q_tiles - 1 - at.rank;
  const int b = bh / p.Hq, h = bh - b * p.Hq, hk = h / p.group;
  const Sample sample = sample_of(p, b);
  const int klen = sample.keys, first = sample.first, prefix = sample.prefix;
  const int row0 = tile * 128 + 32 * wave, rows = min(p.Sq - row0, 32), i = row0 + j32;
  const bool docs = p.docs_q != nullptr;
  const int nqb = (p.Sq + kBlock - 1) / kBlock, nkb = (p.Sk + kBlock - 1) / kBlock;

  LaneRow L;
  L.pos = first + i;
  L.limit = row_limit(p.causal, klen, prefix, L.pos);
  L.doc = docs ? doc_at(p.docs_q, (int64_t)b * p.Sq + i, i < p.Sq, -1) : 0;
  L.slope = BIAS == kBiasSlopes ? p.slopes[h] * p.slope_mul : 0.f;
  L.tab = tab;
  floatx2_t st = {INFINITY, 0.f};
  if (i < p.Sq) st = bp.stats[(int64_t)bh * (64 * nqb) + i];
  const float lse = st[0], delta = st[1];
  // Q^T and dO^T as B operands; rows without keys are zeros, whatever the tensors hold there
  half8_t qf[D / 16], df[D / 16];
  {
    const int ic = min(i, p.Sq - 1);
    const half_t* qs = p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)ic * p.qs[2];
    const half_t* ds = bp.dout + b * bp.dos[0] + h * bp.dos[1] + (int64_t)ic * bp.dos[2];
    const bool live = lse != INFINITY;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const half8_t z = {};
      qf[ks] = live ? *reinterpret_cast<const half8_t*>(qs + 16 * ks + 8 * g) : z;
      df[ks] = live ? *reinterpret_cast<const half8_t*>(ds + 16 * ks + 8 * g) : z;
    }
  }
  constexpr float shift = BF ? 0.f : (float)kPShift;
  float up = 1.f, down = bp.scale;              // fp16: dT is formed times 2^kPShift (as P is) and carried times 2^k
  if constexpr (!BF) {
    float m = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, __builtin_fabsf((float)df[ks][e]));
    const int k = dt_shift<D>(pair_max(m), wave_max_of(bp.vmax + ((int64_t)b * p.Hkv + hk) * nkb, nkb));
    up = pow2(k - kPShift);
    down = bp.scale * pow2(-k);
  }

  TileSource<D, kBlock> ksrc, vsrc;
  ksrc.set(p.k + b * p.ks[0] + hk * p.ks[1], p.ks[2]);
  vsrc.set(p.v + b * p.vs[0] + hk * p.vs[1], p.vs[2]);
  uint32_t k_off[TL::kN], v_off[TL::kN];
  TL::offsets(k_off, wave, lane, p.ks[2]);
  TL::offsets(v_off, wave, lane, p.vs[2]);
  int rd[D / 16], tr[D / 32][2];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) rd[ks] = frag_off<D>(j32, g, ks);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) tr[dt][hh] = tr_off<D>(lane, dt, hh);

  const int wg_rows = min(p.Sq - tile * 128, 128);
  const int wg_hi = row_limit(p.causal, klen, prefix, first + tile * 128 + wg_rows - 1);
  const int my_hi = rows > 0 ? row_limit(p.causal, klen, prefix, first + row0 + rows - 1) : 0;
  const int my_lo = rows > 0 ? row_limit(p.causal, klen, prefix, first + row0) : 0;
  DocRange qa = {0, 0, 1, 0}, qb = qa;
  if (docs) {
    const DocRange* dr = p.dr_q + (int64_t)b * nqb + 2 * tile;
    qa = dr[0];
    qb = 2 * tile + 1 < nqb ? dr[1] : DocRange{1, 0, 0, 0};
  }
  const DocRange mine = wave < 2 ? qa : qb;
  const int n_win = ((wg_hi + kBlock - 1) / kBlock + 63) >> 6;
  uint64_t set_load = 0, set_mine = 0, set_full = 0;
  auto window = [&](int w) {
    const int t = 64 * w + lane, j0 = t * kBlock;
    bool load = j0 < wg_hi, own = j0 < my_hi, full = j0 + kBlock <= my_lo;
    if (docs && load) {
      const DocRange r = p.dr_k[(int64_t)b * nkb + t];
      const bool ia = ranges_meet(r, qa), ib = ranges_meet(r, qb);
      load = ia || ib;
      own = own && (wave < 2 ? ia : ib);
      full = full && ranges_one(r, mine);
    }
    set_load = __ballot(load); set_mine = __ballot(own); set_full = __ballot(full);
  };
  struct Step { int t; int mine; int full; };
  int win = 0;
  if (n_win > 0) window(0);
  auto next_step = [&]() -> Step {
    while (set_load == 0) {
      if (++win >= n_win) return Step{-1, 0, 0};
      window(win);
    }
    const int bit = __builtin_ctzll(set_load);
    set_load &= set_load - 1;
    return Step{64 * win + bit, (int)((set_mine >> bit) & 1), (int)((set_full >> bit) & 1)};
  };

  floatx16 acc[D / 32], mac[D / 32];            // dT K and M
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) { acc[x][r] = 0.f; mac[x][r] = 0.f; }
  float off = 0.f;                              // delta' - delta: sum_j P_ij (dP_ij - delta) (this lane's keys)

  int next_valid = 0, next_id = 0;
  auto issue = [&](int t, lds_byte* kd, lds_byte* vd) {
    const int valid = min(klen - t * kBlock, kBlock);
    // (the loaded id as it is: anything computed from it here would wait for the load)
    if (docs) next_id = p.docs_k[(int64_t)b * p.Sk + t * kBlock + min(lane, valid - 1)];
    next_valid = valid;
    TL::issue(ksrc.tile(t, valid), k_off, wave, kd);
    TL::issue(vsrc.tile(t, valid), v_off, wave, vd);
  };
  auto step = [&](const Step cur, const Step nxt, lds_byte* kt, lds_byte* vt, lds_byte* kn, lds_byte* vn) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    const int cur_id = lane < next_valid ? doc_or(next_id, -2) : -2;
    if (docs) {
      const uint64_t valid = __ballot(cur_id >= 0);
      if (~valid) { TL::keep(valid, wave, lane, kt); TL::keep(valid, wave, lane, vt); }
    }
    __syncthreads();
    if (nxt.t >= 0) issue(nxt.t, kn, vn);
    if (!cur.mine) return;
    if (docs && !cur.full) {
      doc_ids[wave][lane] = cur_id;
      __builtin_amdgcn_wave_barrier();
    }
    constexpr bool PIPE = D == 128;
    typedef Phases<PIPE> PH;
    constexpr int NK = D / 16, kEl = 16 / NK;      // slices per phase, scores per slice of softmax
    half8_t ring[3][2];
    auto fetch = [&](int n) {
      const int ph = n / NK, i = n % NK, off = 32 * PH::piece(ph) * (2 * D);
      if (ph < 4 && PH::scores(ph)) {
        ring[n % 3][0] = lds_frag(kt + off + rd[i]);
        ring[n % 3][1] = lds_frag(vt + off + rd[i]);
      } else if (ph < 4) {
        ring[n % 3][0] = frag_tr<D>(kt + off, i, tr);
      }
    };
    floatx16 s[2] = {zero16(), zero16()}, dp[2] = {zero16(), zero16()}, w[2];
    half8_t x[2][2], y[2][2];
    float cc[2] = {p.cc, p.cc}, add[2] = {0.f, 0.f};
    auto softmax = [&](int mt, int r) {
      float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r], cc[mt], shift - lse + add[mt]));
      float d = pr * (dp[mt][r] - delta);
      off += d;
      if constexpr (CAP) { d *= w[mt][r]; pr *= w[mt][r]; }
      x[mt][r >> 3][r & 7] = to_elem<BF>(BF ? d : d * up);
      y[mt][r >> 3][r & 7] = to_elem<BF>(pr);
    };
    auto rule = [&](int mt) {
      const int j0 = cur.t * kBlock + 32 * mt + 4 * g;
      if constexpr (CAP) cap_scores_grad(p, s[mt], w[mt]);
      bool look_up = true;
      if constexpr (BIAS == kBiasTable) {
        const int at = cur.t * kBlock + 32 * mt - (first + row0);
        const FarPiece f = far_piece(p, tab, at - 31, at + 31);
        if (f.far) { look_up = false; cc[mt] = p.c; add[mt] = f.add; }
      }
      if (look_up) bias_scores<BIAS>(p, L, j0, s[mt]);
      if (!cur.full) {
        limit_scores(L, j0, s[mt]);
        if (docs) doc_scores(L, &doc_ids[wave][32 * mt + 4 * g], s[mt]);
      }
    };
    fetch(0);
    fetch(1);
    auto phase = [&](auto number) {
      constexpr int ph = decltype(number)::value, mt = PH::piece(ph);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int n = ph * NK + i;
        fetch(n + 2);
        STOF_FENCE();
        if constexpr (PH::scores(ph)) {
          s[mt] = mfma32<BF>(ring[n % 3][0], qf[i], s[mt]);
          dp[mt] = mfma32<BF>(ring[n % 3][1], df[i], dp[mt]);
        } else {
          const int s2 = i / (D / 32), dt = i % (D / 32);
          mac[dt] = mfma32<BF>(ring[n % 3][0], y[mt][s2], mac[dt]);
          acc[dt] = mfma32<BF>(ring[n % 3][0], x[mt][s2], acc[dt]);
        }
        if constexpr (PIPE && (ph == 1 || ph == 2)) {
#pragma unroll
          for (int e = 0; e < kEl; ++e) softmax(ph - 1, kEl * i + e);
        }
        STOF_FENCE();
      }
      if constexpr (PH::scores(ph)) {
        rule(mt);
        if constexpr (!PIPE) {
#pragma unroll
          for (int r = 0; r < 16; ++r) softmax(mt, r);
        }
      }
    };
    phase(std::integral_constant<int, 0>());
    phase(std::integral_constant<int, 1>());
    phase(std::integral_constant<int, 2>());
    phase(std::integral_constant<int, 3>());
  };
  Step cur = next_step();
  if (cur.t >= 0) issue(cur.t, (lds_byte*)k0, (lds_byte*)v0);
  if constexpr (BIAS == kBiasTable) load_table<BF>(p, h, tab, threadIdx.x, 256);   // (the walk's first barrier covers it)
  while (cur.t >= 0) {
    Step nxt = next_step();
    step(cur, nxt, (lds_byte*)k0, (lds_byte*)v0, (lds_byte*)k1, (lds_byte*)v1);
    cur = nxt;
    if (nxt.t >= 0) {
      cur = next_step();
      step(nxt, cur, (lds_byte*)k1, (lds_byte*)v1, (lds_byte*)k0, (lds_byte*)v0);
    }
  }
  __syncthreads();
  if (rows <= 0) return;
  off = pair_sum(off) * (BF ? 1.f : pow2(-kPShift));
  if (g == 0 && i < p.Sq && lse != INFINITY) bp.stats[(int64_t)bh * (64 * nqb) + i][1] = delta + off;
  // both terms to the scale of the output: dT K by `down`, M (carried times 2^kPShift in fp16) by the row's difference
  const float fix = -off * bp.scale * (BF ? 1.f : pow2(-kPShift));
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[x][r] = __builtin_fmaf(acc[x][r], down, mac[x][r] * fix);
  lds_byte* stage = (lds_byte*)(wave == 0 ? k0 : wave == 1 ? k1 : wave == 2 ? v0 : v1);
  store_rows<D, BF>(acc, 1.f, stage, bp.dq + ((int64_t)bh * p.Sq + row0) * D, rows, lane);
}

// d table[h][x]: the workgroups' sums over batch and key tiles, in order.  Sixteen slices of them per entry.
template <bool BF>
__global__ __launch_bounds__(1024) void score_attn_bwd_table_kernel(const BwdParams bp) {
  const ScoreParams& p = bp.s;
  __shared__ float part[16][64];
  const int n_dist = 2 * p.radius + 1;
  const int h = blockIdx.y, x = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
  const int tiles = bp.k_tiles * bp.splits, n = p.B * tiles, per = (n + 15) / 16;
  float t = 0.f;                   // (fp16: carried times 2^kPShift)
  if (x < n_dist) {
#pragma unroll 4
    for (int y = slice * per; y < min(n, (slice + 1) * per); ++y) {
      const int b = y / tiles, tile = y - b * tiles;
      t += bp.tab_part[(((int64_t)b * p.Hq + h) * tiles + tile) * n_dist + x];
    }
  }
  part[slice][threadIdx.x & 63] = t;
  __syncthreads();
  if (slice == 0 && x < n_dist) {
    float sum = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) sum += part[y][threadIdx.x];
    bp.dtable[(int64_t)h * n_dist + x] = to_elem<BF>((BF ? 1.f : pow2(-kPShift)) * sum);
  }
}

// ---- keys: dK and dV.  128 keys of one key head per workgroup, 32 per wave; walks the query tiles of the heads that
// share it.  Lane = key; the rows' lse and delta come four at a time from the wave's copy in LDS.
//
// Table (TAB): the dS of a 32 x 32 piece go through LDS (fp32, row pitch 33: lane l then reads diagonal l - 31, 32
// consecutive words per step for the wave, no conflicts) and every diagonal's sum is added by one lane to
// the wave's own array; diagonals that clip, and pieces that lie beyond the radius as a whole, are
// added in two registers per lane.  After each head the waves' arrays are joined and written to the
// workspace, which a last kernel adds up over batch and key tiles.
//
// Bound: LDS reads beside MFMA and vector issue (both operands of the sums' products are transposed on the way; 1.8 to 2.1 reads
// per MFMA).  bf16, B2 H16 S2048: D64 90 us (760 TFLOP/s, MFMA busy 43 %), with a table 112; D128 157 us (875 TFLOP/s, 41 %), table 190.
template <int D, bool BF, bool CAP, int BIAS>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void score_attn_bwd_k_kernel(const BwdParams bp) {
  const ScoreParams& p = bp.s;
  typedef TileLoad<D, kBlock, 4> TL;
  __shared__ __attribute__((aligned(1024))) unsigned char q0[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char q1[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char d0[TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char d1[TL::kBytes];
  __shared__ int doc_ids[4][kBlock];
  __shared__ __attribute__((aligned(16))) float st_lse[4][kBlock];
  __shared__ __attribute__((aligned(16))) float st_del[4][kBlock];
  constexpr bool TAB = BIAS == kBiasTable;
  __shared__ float skew[TAB ? 4 : 1][TAB ? 32 + 32 * 33 + 32 : 1];
  extern __shared__ float tab[];                // kBiasTable: the head's table, then 2 R + 1 sums per wave

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;
  Placed at;
  if (!place(blockIdx.x, p.B * p.Hkv, 1, bp.k_tiles * bp.splits, bp.k_chunk, p.cus_per_xcd, D == 64 ? 2 : 1, p.causal, p.uneven != kEven ? kUnevenTiles : kEven, at)) return;
  const int bk = at.head, slot = at.rank;
  const int tile = slot / bp.splits, split = slot - tile * bp.splits;   // (causal: the first keys have most queries)
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const Sample sample = sample_of(p, b);
  const int klen = sample.keys, first = sample.first, prefix = sample.prefix;
  const int key0 = tile * 128 + 32 * wave, keys = min(p.Sk - key0, 32), j = key0 + j32;
  const bool docs = p.docs_q != nullptr;
  const int nqb = (p.Sq + kBlock - 1) / kBlock, nkb = (p.Sk + kBlock - 1) / kBlock;
  const int doc = docs ? doc_at(p.docs_k, (int64_t)b * p.Sk + j, j < klen, -2) : 0;
  const bool live = j < klen && doc >= 0;
  // queries at positions >= from see this key
  const int from = !live ? (1 << 30) : (p.causal && j >= prefix) ? j : -(1 << 30);

  half8_t kf[D / 16], vf[D / 16];
  {
    const int jc = min(j, p.Sk - 1);
    const half_t* ks_ = p.k + b * p.ks[0] + hk * p.ks[1] + (int64_t)jc * p.ks[2];
    const half_t* vs_ = p.v + b * p.vs[0] + hk * p.vs[1] + (int64_t)jc * p.vs[2];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const half8_t z = {};
      kf[ks] = live ? *reinterpret_cast<const half8_t*>(ks_ + 16 * ks + 8 * g) : z;
      vf[ks] = live ? *reinterpret_cast<const half8_t*>(vs_ + 16 * ks + 8 * g) : z;
    }
  }
  float up = 1.f, down = bp.scale;
  if constexpr (!BF) {
    // (the head's largest |V|, not the lane's own key's: a heavily attended key of small values has the delta of the others')
    const int k = dt_shift<D>(wave_max_of(bp.domax + ((int64_t)b * p.Hq + hk * p.group) * nqb, p.group * nqb),
                              wave_max_of(bp.vmax + ((int64_t)b * p.Hkv + hk) * nkb, nkb));
    up = pow2(k - kPShift);
    down = bp.scale * pow2(-k);
  }

  uint32_t q_off[TL::kN], d_off[TL::kN];
  TL::offsets(q_off, wave, lane, p.qs[2]);
  TL::offsets(d_off, wave, lane, bp.dos[2]);
  int rd[D / 16], tr[D / 32][2];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) rd[ks] = frag_off<D>(j32, g, ks);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) tr[dt][hh] = tr_off<D>(lane, dt, hh);

  DocRange ka = {0, 0, 1, 0}, kc = ka;
  if (docs) {
    const DocRange* dr = p.dr_k + (int64_t)b * nkb + 2 * tile;
    ka = dr[0];
    kc = 2 * tile + 1 < nkb ? dr[1] : DocRange{1, 0, 0, 0};
  }
  const DocRange mine = wave < 2 ? ka : kc;
  const int wg_key = tile * 128;
  const int n_win = wg_key < klen ? (nqb + 63) >> 6 : 0;
  uint64_t set_load = 0, set_mine = 0, set_full = 0;
  auto window = [&](int w) {
    const int t = 64 * w + lane, hi = first + min(64 * t + 63, p.Sq - 1), lo = first + 64 * t;   // positions of the tile
    const bool in = t < nqb && t % bp.splits == split;
    bool load = in && (!p.causal || hi >= wg_key || wg_key < prefix);
    bool own = in && key0 < klen && (!p.causal || hi >= key0 || key0 < prefix);
    bool full = key0 + 32 <= klen && (!p.causal || lo >= key0 + 31 || key0 + 32 <= prefix);
    if (docs && load) {
      const DocRange r = p.dr_q[(int64_t)b * nqb + t];
      const bool ia = ranges_meet(r, ka), ib = ranges_meet(r, kc);
      load = ia || ib;
      own = own && (wave < 2 ? ia : ib);
      full = full && ranges_one(r, mine);
    }
    set_load = __ballot(load); set_mine = __ballot(own); set_full = __ballot(full);
  };
  struct Step { int t; int head; int mine; int full; };
  int win = 0, hg = 0;
  if (n_win > 0) window(0);
  auto next_step = [&]() -> Step {
    while (set_load == 0) {
      if (++win >= n_win) {
        win = 0;
        if (n_win == 0 || ++hg >= p.group) return Step{-1, 0, 0, 0};
      }
      window(win);
    }
    const int bit = __builtin_ctzll(set_load);
    set_load &= set_load - 1;
    return Step{64 * win + bit, hg, (int)((set_mine >> bit) & 1), (int)((set_full >> bit) & 1)};
  };

  floatx16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[x][r] = 0.f; dv[x][r] = 0.f; }

  LaneRow L;                       // (distances run the other way here: see below)
  L.slope = 0.f; L.tab = tab; L.pos = 0; L.limit = 0; L.doc = doc;
  int table_head = -1;
  const int n_dist = 2 * p.radius + 1;
  float* sums = tab + n_dist + 2 * kTabPad + wave * n_dist;   // TAB
  float far_lo = 0.f, far_hi = 0.f;
  // TAB: the sums of head `head`, joined over the waves, to the workspace; all threads, with barriers.  The arrays are zero afterwards.
  auto flush = [&](int head) {
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {          // (radius 0: one entry, both sides)
      sums[0] += far_lo;
      sums[n_dist - 1] += far_hi;
    }
    far_lo = far_hi = 0.f;
    __syncthreads();
    float* all = tab + n_dist + 2 * kTabPad;
    float* part = bp.tab_part + (((int64_t)b * p.Hq + hk * p.group + head) * (bp.k_tiles * bp.splits) + slot) * n_dist;
    for (int x = threadIdx.x; x < n_dist; x += 256) {
      part[x] = (all[x] + all[n_dist + x]) + (all[2 * n_dist + x] + all[3 * n_dist + x]);
      all[x] = all[n_dist + x] = all[2 * n_dist + x] = all[3 * n_dist + x] = 0.f;
    }
    __syncthreads();
  };
  int flushed = 0;                 // heads whose sums are written
  if constexpr (TAB) {
    for (int x = lane; x < n_dist; x += 64) sums[x] = 0.f;
  }
  float slope = 0.f;
  int next_id = 0;
  floatx2_t next_st = {INFINITY, 0.f};
  TileSource<D, kBlock> qsrc, dsrc;
  const floatx2_t* stats = nullptr;
  int issue_head = -1;
  auto issue = [&](const Step& s, lds_byte* qd, lds_byte* dd) {
    const int valid = min(p.Sq - s.t * kBlock, kBlock);
    if (s.head != issue_head) {
      const int h = hk * p.group + s.head;
      issue_head = s.head;
      qsrc.set(p.q + b * p.qs[0] + h * p.qs[1], p.qs[2]);
      dsrc.set(bp.dout + b * bp.dos[0] + h * bp.dos[1], bp.dos[2]);
      stats = bp.stats + ((int64_t)b * p.Hq + h) * (64 * nqb);
    }
    if (docs) next_id = p.docs_q[(int64_t)b * p.Sq + s.t * kBlock + min(lane, valid - 1)];   // (as it is: see the query kernel)
    next_st = stats[s.t * kBlock + lane];
    TL::issue(qsrc.tile(s.t, valid), q_off, wave, qd);
    TL::issue(dsrc.tile(s.t, valid), d_off, wave, dd);
  };
  auto step = [&](const Step cur, const Step nxt, lds_byte* qt, lds_byte* dt_, lds_byte* qn, lds_byte* dn) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    const int cur_id = doc_or(next_id, -1);      // (rows past the end have no lse)
    const floatx2_t cur_st = next_st;
    // rows without keys: zeros, whatever the tensors hold there
    const uint64_t rows = __ballot(cur_st[0] != INFINITY);
    if (~rows) { TL::keep(rows, wave, lane, qt); TL::keep(rows, wave, lane, dt_); }
    if (TAB && cur.head != table_head) {
      if constexpr (TAB)
        for (; flushed < cur.head; ++flushed) flush(flushed);
      __syncthreads();             // every wave is done with the previous head's table
      load_table<BF>(p, hk * p.group + cur.head, tab, threadIdx.x, 256);
      table_head = cur.head;
    }
    if constexpr (BIAS == kBiasSlopes) slope = p.slopes[hk * p.group + cur.head] * p.slope_mul;
    __syncthreads();
    if (nxt.t >= 0) issue(nxt, qn, dn);
    if (!cur.mine) return;
    FarPiece far[2] = {};
    if constexpr (TAB) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int d_lo = key0 - (first + cur.t * kBlock + 32 * mt) - 31;
        far[mt] = far_piece(p, tab, d_lo, d_lo + 62);
      }
    }
    st_lse[wave][lane] = cur_st[0] - (BF ? 0.f : (float)kPShift) - (g ? far[1].add : far[0].add);   // fp16: P comes out times 2^kPShift
    st_del[wave][lane] = cur_st[1];
    if (docs && !cur.full) doc_ids[wave][lane] = cur_id;
    __builtin_amdgcn_wave_barrier();
    constexpr bool PIPE = D == 128 && !TAB;
    typedef Phases<PIPE> PH;
    constexpr int NK = D / 16, kEl = 16 / NK;
    half8_t ring[3][2];
    auto fetch = [&](int n) {
      const int ph = n / NK, i = n % NK, off = 32 * PH::piece(ph) * (2 * D);
      if (ph < 4 && PH::scores(ph)) {
        ring[n % 3][0] = lds_frag(qt + off + rd[i]);
        ring[n % 3][1] = lds_frag(dt_ + off + rd[i]);
      } else if (ph < 4) {
        ring[n % 3][0] = frag_tr<D>(dt_ + off, i, tr);
        ring[n % 3][1] = frag_tr<D>(qt + off, i, tr);
      }
    };
    floatx16 s[2] = {zero16(), zero16()}, dp[2] = {zero16(), zero16()}, w[2];
    half8_t x[2][2], y[2][2];                       // dT and P
    floatx4 ls, de;
    auto softmax = [&](int mt, int r) {
      if (r % 4 == 0) {
        ls = *reinterpret_cast<const floatx4*>(&st_lse[wave][32 * mt + 2 * r + 4 * g]);
        de = *reinterpret_cast<const floatx4*>(&st_del[wave][32 * mt + 2 * r + 4 * g]);
      }
      const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r], TAB && far[mt].far ? p.c : p.cc, -ls[r % 4]));
      y[mt][r >> 3][r & 7] = to_elem<BF>(pr);
      float d = pr * (dp[mt][r] - de[r % 4]);
      if constexpr (TAB) s[mt][r] = d;
      if constexpr (CAP) d *= w[mt][r];
      x[mt][r >> 3][r & 7] = to_elem<BF>(BF ? d : d * up);
    };
    auto rule = [&](int mt) {
      const int pos0 = first + cur.t * kBlock + 32 * mt + 4 * g;    // position of the lane's score 0; score r: + key_off(r)
      if constexpr (CAP) cap_scores_grad(p, s[mt], w[mt]);
      if constexpr (TAB) {
        if (!far[mt].far) {
          const int at = min(max(j - pos0, -p.radius), p.radius + kTabPad);   // distance j - p falls with the row
          const float* t = tab + (at + p.radius + kTabPad);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[mt][r] = __builtin_fmaf(s[mt][r], p.c, t[-key_off(r)]);
        }
      } else if constexpr (BIAS == kBiasSlopes) {
        const float at = (float)(j - pos0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mt][r] = __builtin_fmaf(__builtin_fabsf(at - (float)key_off(r)), -slope, s[mt][r]);
      }
      if (!cur.full) {
        const int rel = from - pos0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[mt][r] = key_off(r) >= rel ? s[mt][r] : -INFINITY;
        if (docs) doc_scores(L, &doc_ids[wave][32 * mt + 4 * g], s[mt]);
      }
    };
    // TAB: piece mt's dS (in s) to the sums of the distances
    auto distances = [&](int mt) {
      const int d_lo = key0 - (first + cur.t * kBlock + 32 * mt) - 31, d_hi = d_lo + 62;   // distances of the piece
      if (d_lo >= p.radius || d_hi <= -p.radius) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += s[mt][r];
        if (d_lo >= p.radius) far_hi += t; else far_lo += t;
      } else {
        float* sk = skew[wave] + 32;            // [query][key], row pitch 33, room on both sides
#pragma unroll
        for (int r = 0; r < 16; ++r) sk[(key_off(r) + 4 * g) * 33 + j32] = s[mt][r];
        __builtin_amdgcn_wave_barrier();
        int dg = lane - 31;                     // lane l sums the diagonal key - query = l - 31 of the piece
        asm volatile("" : "+v"(dg));            // (or the 32 predicates below are kept across the walk, in spilled registers)
        const float* at = sk + dg;
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const float e = at[34 * q];
          t += (unsigned)(q + dg) < 32u ? e : 0.f;
        }
        __builtin_amdgcn_wave_barrier();
        if (lane < 63) {
          const int d = d_lo + lane;
          if (d >= p.radius) far_hi += t;
          else if (d <= -p.radius) far_lo += t;
          else sums[d + p.radius] += t;
        }
      }
    };
    fetch(0);
    fetch(1);
    auto phase = [&](auto number) {
      constexpr int ph = decltype(number)::value, mt = PH::piece(ph);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int n = ph * NK + i;
        fetch(n + 2);
        STOF_FENCE();
        if constexpr (PH::scores(ph)) {
          s[mt] = mfma32<BF>(ring[n % 3][0], kf[i], s[mt]);
          dp[mt] = mfma32<BF>(ring[n % 3][1], vf[i], dp[mt]);
        } else {
          const int s2 = i / (D / 32), dt = i % (D / 32);
          dv[dt] = mfma32<BF>(ring[n % 3][0], y[mt][s2], dv[dt]);
          dk[dt] = mfma32<BF>(ring[n % 3][1], x[mt][s2], dk[dt]);
        }
        if constexpr (PIPE && (ph == 1 || ph == 2)) {
#pragma unroll
          for (int e = 0; e < kEl; ++e) softmax(ph - 1, kEl * i + e);
        }
        STOF_FENCE();
      }
      if constexpr (PH::scores(ph)) {
        rule(mt);
        if constexpr (!PIPE) {
#pragma unroll
          for (int r = 0; r < 16; ++r) softmax(mt, r);
          if constexpr (TAB) distances(mt);
        }
      }
    };
    phase(std::integral_constant<int, 0>());
    phase(std::integral_constant<int, 1>());
    phase(std::integral_constant<int, 2>());
    phase(std::integral_constant<int, 3>());
  };
  Step cur = next_step();
  if (cur.t >= 0) issue(cur, (lds_byte*)q0, (lds_byte*)d0);
  while (cur.t >= 0) {
    Step nxt = next_step();
    step(cur, nxt, (lds_byte*)q0, (lds_byte*)d0, (lds_byte*)q1, (lds_byte*)d1);
    cur = nxt;
    if (nxt.t >= 0) {
      cur = next_step();
      step(nxt, cur, (lds_byte*)q1, (lds_byte*)d1, (lds_byte*)q0, (lds_byte*)d0);
    }
  }
  if constexpr (TAB)
    for (; flushed < p.group; ++flushed) flush(flushed);
  __syncthreads();
  if (keys <= 0) return;
  lds_byte* stage = (lds_byte*)(wave == 0 ? q0 : wave == 1 ? q1 : wave == 2 ? d0 : d1);
  const int64_t row = ((int64_t)bk * p.Sk + key0) * D;
  if (bp.splits > 1) {
    if (j32 >= keys) return;
    const int64_t n = (int64_t)p.B * p.Hkv * p.Sk * D;
    float* ok = bp.kv_part + split * n + row + j32 * D;
    float* ov = ok + bp.splits * n;
    const float mul_v = BF ? 1.f : pow2(-kPShift);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        floatx4 a, c;
#pragma unroll
        for (int e = 0; e < 4; ++e) { a[e] = dk[dt][4 * q4 + e] * down; c[e] = dv[dt][4 * q4 + e] * mul_v; }
        *reinterpret_cast<floatx4*>(ok + 32 * dt + 8 * q4 + 4 * g) = a;
        *reinterpret_cast<floatx4*>(ov + 32 * dt + 8 * q4 + 4 * g) = c;
      }
    return;
  }
  store_rows<D, BF>(dk, down, stage, bp.dk + row, keys, lane);
  store_rows<D, BF>(dv, BF ? 1.f : pow2(-kPShift), stage, bp.dv + row, keys, lane);
}

// dK and dV from the sums of the splits, in their order; eight values per thread.
template <bool BF>
__global__ __launch_bounds__(256) void score_attn_bwd_join_kernel(const float* part, half_t* dk, half_t* dv, int64_t n, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= 2 * n) return;
  const bool v = i >= n;
  const int64_t at = v ? i - n : i;
  const float* src = part + (v ? splits * n : 0) + at;
  floatx4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
  for (int s = 0; s < splits; ++s) {
    a += *reinterpret_cast<const floatx4*>(src + s * n);
    b += *reinterpret_cast<const floatx4*>(src + s * n + 4);
  }
  half8_t o;
#pragma unroll
  for (int e = 0; e < 4; ++e) { o[e] = to_elem<BF>(a[e]); o[4 + e] = to_elem<BF>(b[e]); }
  *reinterpret_cast<half8_t*>((v ? dv : dk) + at) = o;
}

// ---- host side

// Workgroups per key tile: few key heads (shared by many query heads) and short sequences leave the device
// empty while each workgroup walks all their query tiles.  Up to 256 workgroups, split s takes every splits-th query
// tile, until 512 workgroups (two per compute unit) have work of at least four tiles each; their fp32 sums are
// joined by one more kernel.  B2 H16/4 S2048 D128 causal, 128 workgroups: 246 us unsplit, 103 + 12 us with four
// splits; B8 H12 S512 D64 with a table, 384 workgroups: 51 + 4 us unsplit, 44 + 18 us with two.
int key_splits(int B, int Hkv, int Sq, int Sk, int group) {
  const int64_t wgs = (int64_t)B * Hkv * ((Sk + 127) / 128);
  const int64_t want = 512;
  const int most = ((Sq + 63) / 64 * group + 3) / 4;
  int64_t n = wgs > want / 2 ? 1 : (want + wgs - 1) / wgs;
  if (n > (Sq + 63) / 64) n = (Sq + 63) / 64;
  if (n > most) n = most;
  return n > 8 ? 8 : (int)n;
}

struct Layout { int64_t stats, domax, vmax, part, kv, total; };

Layout layout(int B, int Hq, int Hkv, int Sq, int Sk, int D, int radius, int docs) {
  const int64_t nq = (Sq + 63) / 64, nk = (Sk + 63) / 64, kt = (Sk + 127) / 128;
  auto up = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
  Layout l;
  l.stats = docs ? up((int64_t)B * (nq + nk) * (int64_t)sizeof(DocRange)) : 0;
  l.domax = l.stats + up((int64_t)B * Hq * nq * 64 * 8);
  l.vmax = l.domax + up((int64_t)B * Hq * nq * 4);
  l.part = l.vmax + up((int64_t)B * Hkv * nk * 4);
  const int splits = key_splits(B, Hkv, Sq, Sk, Hq / Hkv);
  l.kv = l.part + (radius >= 0 ? up((int64_t)B * Hq * kt * splits * (2 * radius + 1) * 4) : 0);
  l.total = l.kv + (splits > 1 ? 2 * splits * up((int64_t)B * Hkv * Sk * D * 4) : 0);
  return l;
}

template <int D, bool BF, bool CAP, int BIAS>
void launch_main(BwdParams& p, hipStream_t st) {
  const int n_dist = BIAS == kBiasTable ? 2 * p.s.radius + 1 : 0, n_tab = BIAS == kBiasTable ? n_dist + 2 * kTabPad : 0;
  const unsigned gq = 8u * (unsigned)p.q_chunk, gk = 8u * (unsigned)p.k_chunk;
  score_attn_bwd_q_kernel<D, BF, CAP, BIAS><<<dim3(gq), dim3(256), (size_t)n_tab * 4, st>>>(p);
  score_attn_bwd_k_kernel<D, BF, CAP, BIAS><<<dim3(gk), dim3(256), (size_t)(n_tab + 4 * n_dist) * 4, st>>>(p);
}
template <int D, bool BF, bool CAP>
void launch_bias(BwdParams& p, hipStream_t st) {
  if (p.s.table) launch_main<D, BF, CAP, kBiasTable>(p, st);
  else if (p.s.slopes) launch_main<D, BF, CAP, kBiasSlopes>(p, st);
  else launch_main<D, BF, CAP, kBiasNone>(p, st);
}
template <int D, bool BF>
void launch_bwd(BwdParams& p, hipStream_t st) {
  const ScoreParams& s = p.s;
  const int nq = (s.Sq + 63) / 64, nk = (s.Sk + 63) / 64;
  score_attn_bwd_prep_kernel<D, BF><<<dim3((unsigned)(s.B * s.Hq * nq + (BF ? 0 : s.B * s.Hkv * nk) + (p.ranges + 3) / 4)), dim3(256), 0, st>>>(p);
  s.k1 != 0.f ? launch_bias<D, BF, true>(p, st) : launch_bias<D, BF, false>(p, st);
  if (p.splits > 1) {
    const int64_t n = (int64_t)s.B * s.Hkv * s.Sk * D;
    score_attn_bwd_join_kernel<BF><<<dim3((unsigned)((2 * n / 8 + 255) / 256)), dim3(256), 0, st>>>(p.kv_part, p.dk, p.dv, n, p.splits);
  }
  if (s.table)
    score_attn_bwd_table_kernel<BF><<<dim3((unsigned)((2 * s.radius + 64) / 64), (unsigned)s.Hq), dim3(1024), 0, st>>>(p);
}

}  // namespace

extern "C" int64_t stof_score_attn_bwd_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Sk, int D, int radius, int docs) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sk <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
  return layout(B, Hq, Hkv, Sq, Sk, D, radius, docs).total;
}

extern "C" int stof_score_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse,
                                   void* dq, void* dk, void* dv, void* dtable,
                                   const void* table, const float* slopes, const int32_t* prefix, const int32_t* kv_len,
                                   const int32_t* docs_q, const int32_t* docs_k,
                                   float scale, float cap, int radius, int causal, int q_start, int q_end,
                                   const int64_t* dout_strides, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* out_strides, int B, int Hq, int Hkv, int Sq, int Sk, int D, int dtype,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  const void* req[] = {dout, q, k, v, out, lse, dq, dk, dv, workspace};
  const int64_t* str[] = {dout_strides, q_strides, k_strides, v_strides, out_strides};
  const int rc = score_attn_check(req, 10, str, 5, B, Hq, Hkv, Sq, Sk, D, dtype, scale, cap, table ? radius : -1);
  if (rc) return rc;
  if (Sk == 0) return STOF_ERR_BAD_SHAPE;
  if (table && slopes) return STOF_ERR_UNSUPPORTED;
  if (table && radius < 0) return STOF_ERR_BAD_SHAPE;
  if (table && !dtable) return STOF_ERR_NULL_POINTER;
  if ((docs_q == nullptr) != (docs_k == nullptr)) return STOF_ERR_NULL_POINTER;
  if (q_end && !kv_len) return STOF_ERR_NULL_POINTER;
  if (q_start > (1 << 29) || q_start < -(1 << 29)) return STOF_ERR_BAD_SHAPE;
  const Layout l = layout(B, Hq, Hkv, Sq, Sk, D, table ? radius : -1, docs_q != nullptr);
  if (workspace_bytes < l.total) return STOF_ERR_BAD_SHAPE;
  BwdParams p = {};
  score_attn_params(p.s, q, k, v, table, slopes, prefix, kv_len, docs_q, docs_k, scale, cap, radius, causal, q_start, q_end,
                    q_strides, k_strides, v_strides, B, Hq, Hkv, Sq, Sk);
  p.dout = (const half_t*)dout; p.o = (const half_t*)out; p.lse = lse;
  for (int j = 0; j < 3; ++j) { p.dos[j] = dout_strides[j]; p.oos[j] = out_strides[j]; }
  p.dq = (half_t*)dq; p.dk = (half_t*)dk; p.dv = (half_t*)dv; p.dtable = (half_t*)dtable;
  char* ws = (char*)workspace;
  p.stats = (floatx2_t*)(ws + l.stats); p.domax = (float*)(ws + l.domax); p.vmax = (float*)(ws + l.vmax); p.tab_part = (float*)(ws + l.part);
  p.scale = scale;
  p.q_tiles = (Sq + 127) / 128; p.k_tiles = (Sk + 127) / 128;
  p.q_chunk = (B * Hq * p.q_tiles + 7) / 8;
  p.splits = key_splits(B, Hkv, Sq, Sk, Hq / Hkv);
  p.kv_part = (float*)(ws + l.kv);
  p.k_chunk = (B * Hkv * p.k_tiles * p.splits + 7) / 8;
  hipStream_t st = (hipStream_t)stream;
  // The backward kernels, one or two workgroups per unit, also gain from spreading documents of key heads that divide (mean
  // of three: B2 H16/4 S2048 D128 138 | 133 us, B8 H12 S1024 D64 84 | 68), unless each XCD gets the same heads of every sample.
  if (docs_q && Hkv % 8 != 0) p.s.uneven = Hq % 8 == 0 ? kUnevenHeads : kUnevenTiles;
  p.ranges = docs_q ? score_attn_ranges_at(p.s, ws) : 0;
  if (D == 64) { if (dtype == STOF_DTYPE_BF16) launch_bwd<64, true>(p, st); else launch_bwd<64, false>(p, st); }
  else { if (dtype == STOF_DTYPE_BF16) launch_bwd<128, true>(p, st); else launch_bwd<128, false>(p, st); }
  return stof_check_launch();
}
