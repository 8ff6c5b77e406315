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
// again: |dT| <= 2 D max|dO| max|V| =: bound, and dT 2^k with k = 14 - ceil(log2 bound) stays below 2^15 and
// keeps 11 bits down to 2^-29 of the bound.  P is carried as 2^12 P.  bfloat16 needs neither.
#include "score_attn.h"

namespace {

struct BwdParams {
  ScoreParams s;
  const half_t* dout; const half_t* o; const float* lse;
  int64_t dos[3], oos[3];
  half_t* dq; half_t* dk; half_t* dv;        // contiguous [B, Hq, Sq, D], [B, Hkv, Sk, D]
  floatx2_t* stats;                          // [B, Hq, 64 ceil(Sq / 64)]: (lse in log2 units, delta); +inf = a row without keys or past the end
  float* vmax; float* domax;                 // fp16: largest |V| per (b, hk, key block), largest |dO| per (b, h, query block)
  float* tab_part; half_t* dtable;           // per workgroup of the query kernel: sums of the 2 R + 1 distances
  float scale;
  int q_tiles, k_tiles, q_chunk, k_chunk;
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
// Grid: B Hq ceil(Sq / 64) workgroups of query rows, then (fp16) B Hkv ceil(Sk / 64) of value rows.
template <int D, bool BF>
__global__ __launch_bounds__(256) void score_attn_bwd_prep_kernel(const BwdParams p) {
  const ScoreParams& s = p.s;
  constexpr int kC = D / 8;                       // lanes per row
  constexpr int kR = 64 / kC;                     // rows per wave and pass
  __shared__ float mx_lds[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane % kC;
  const int nq = (s.Sq + 63) / 64, nk = (s.Sk + 63) / 64;
  const bool is_q = (int)blockIdx.x < s.B * s.Hq * nq;
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
      if (c == 0) p.stats[(int64_t)bh * (64 * nq) + r] = floatx2_t{l == -INFINITY ? INFINITY : l * kLog2e, d};
    }
  } else {
    const int idx = blockIdx.x - s.B * s.Hq * nq, bh = idx / nk, t = idx - bh * nk;
    const int b = bh / s.Hkv, h = bh - b * s.Hkv;
    const int klen = sample_keys(s, b);
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
    const float u = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[r] * p.k1));
    w[r] = 4.f * __builtin_fmaf(-u, u, u);
    s[r] = __builtin_fmaf(u, -2.f * p.capl, p.capl);
  }
}

// A operand rows 32 x D of the tile times the lane's vector: 32 x 32 products
template <int D, bool BF>
__device__ __forceinline__ floatx16 product32(const lds_byte* t, const int (&rd)[D / 16], const half8_t (&f)[D / 16]) {
  floatx16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) s = mfma32<BF>(lds_frag(t + rd[ks]), f[ks], s);
  return s;
}
// acc^T += T^T X for 32 rows of the tile: X in the accumulator layout, as 16-bit values
template <int D, bool BF>
__device__ __forceinline__ void accumulate32(floatx16 (&acc)[D / 32], const lds_byte* t, const int (&tr)[D / 32][2], const half8_t (&x)[2]) {
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const lds_byte* p = t + 16 * s2 * (2 * D);
      acc[dt] = mfma32<BF>(lds_frag_tr(p + tr[dt][0], p + tr[dt][1]), x[s2], acc[dt]);
    }
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
template <int D, bool BF>
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
  const int id = (blockIdx.x & 7) * bp.q_chunk + (blockIdx.x >> 3);
  if (id >= p.B * p.Hq * bp.q_tiles) return;
  const int bh = id / bp.q_tiles, tile = bp.q_tiles - 1 - (id - bh * bp.q_tiles);
  const int b = bh / p.Hq, h = bh - b * p.Hq, hk = h / p.group;
  const int klen = sample_keys(p, b), first = sample_first(p, klen), prefix = sample_prefix(p, b);
  const int row0 = tile * 128 + 32 * wave, rows = min(p.Sq - row0, 32), i = row0 + j32;
  const bool docs = p.docs_q != nullptr;
  const int nqb = (p.Sq + kBlock - 1) / kBlock, nkb = (p.Sk + kBlock - 1) / kBlock;

  LaneRow L;
  L.pos = first + i;
  L.limit = row_limit(p.causal, klen, prefix, L.pos);
  L.doc = docs ? doc_at(p.docs_q, (int64_t)b * p.Sq + i, i < p.Sq, -1) : 0;
  L.slope = p.bias_kind == kBiasSlopes ? p.slopes[h] * kLog2e : 0.f;
  L.tab = tab;
  if (p.bias_kind == kBiasTable) load_table<BF>(p, h, tab, threadIdx.x, 256);

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

  const half_t* kb = p.k + b * p.ks[0] + hk * p.ks[1];
  const half_t* vb = p.v + b * p.vs[0] + hk * p.vs[1];
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

  int next_id = 0;
  auto issue = [&](int t, lds_byte* kd, lds_byte* vd) {
    const int valid = min(klen - t * kBlock, kBlock);
    if (docs) next_id = doc_at(p.docs_k, (int64_t)b * p.Sk + t * kBlock + lane, lane < valid, -2);
    TL::issue(rows_rsrc<D>(kb, p.ks[2], (int64_t)t * kBlock, valid), k_off, wave, kd);
    TL::issue(rows_rsrc<D>(vb, p.vs[2], (int64_t)t * kBlock, valid), v_off, wave, vd);
  };
  auto step = [&](const Step cur, const Step nxt, lds_byte* kt, lds_byte* vt, lds_byte* kn, lds_byte* vn) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    const int cur_id = next_id;
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
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int jb = cur.t * kBlock + 32 * mt, j0 = jb + 4 * g;
      floatx16 s = product32<D, BF>(kt + 32 * mt * (2 * D), rd, qf), w;
      const floatx16 dp = product32<D, BF>(vt + 32 * mt * (2 * D), rd, df);
      if (p.k1 != 0.f) cap_scores_grad(p, s, w);
      if (p.bias_kind != kBiasNone) bias_scores(p, L, j0, s);
      if (!cur.full) {
        limit_scores(L, j0, s);
        if (docs) doc_scores(L, &doc_ids[wave][32 * mt + 4 * g], s);
      }
      half8_t x[2], y[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.cc, shift - lse));
        s[r] = pr * (dp[r] - delta);
        off += s[r];
        if (p.k1 != 0.f) { s[r] *= w[r]; pr *= w[r]; }
        x[r >> 3][r & 7] = to_elem<BF>(BF ? s[r] : s[r] * up);
        y[r >> 3][r & 7] = to_elem<BF>(pr);
      }
      accumulate32<D, BF>(mac, kt + 32 * mt * (2 * D), tr, y);
      accumulate32<D, BF>(acc, kt + 32 * mt * (2 * D), tr, x);
    }
  };
  Step cur = next_step();
  if (cur.t >= 0) issue(cur.t, (lds_byte*)k0, (lds_byte*)v0);
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

// d table[h][x]: the workgroups' sums over batch and key tiles, in order.  Four slices of them per entry.
template <bool BF>
__global__ __launch_bounds__(256) void score_attn_bwd_table_kernel(const BwdParams bp) {
  const ScoreParams& p = bp.s;
  __shared__ float part[4][64];
  const int n_dist = 2 * p.radius + 1;
  const int h = blockIdx.y, x = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
  const int n = p.B * bp.k_tiles, per = (n + 3) / 4;
  float t = 0.f;                   // (fp16: carried times 2^kPShift)
  if (x < n_dist)
    for (int y = slice * per; y < min(n, (slice + 1) * per); ++y) {
      const int b = y / bp.k_tiles, tile = y - b * bp.k_tiles;
      t += bp.tab_part[(((int64_t)b * p.Hq + h) * bp.k_tiles + tile) * n_dist + x];
    }
  part[slice][threadIdx.x & 63] = t;
  __syncthreads();
  if (slice == 0 && x < n_dist) {
    const int y = threadIdx.x;
    bp.dtable[(int64_t)h * n_dist + x] = to_elem<BF>((BF ? 1.f : pow2(-kPShift)) * ((part[0][y] + part[1][y]) + (part[2][y] + part[3][y])));
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
template <int D, bool BF, bool TAB>
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
  __shared__ float skew[TAB ? 4 : 1][TAB ? 32 * 33 + 32 : 1];
  extern __shared__ float tab[];                // kBiasTable: the head's table, then 2 R + 1 sums per wave

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;
  const int id = (blockIdx.x & 7) * bp.k_chunk + (blockIdx.x >> 3);
  if (id >= p.B * p.Hkv * bp.k_tiles) return;
  const int bk = id / bp.k_tiles, tile = id - bk * bp.k_tiles;   // (causal: the first keys have most queries)
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const int klen = sample_keys(p, b), first = sample_first(p, klen), prefix = sample_prefix(p, b);
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
    float m = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, __builtin_fabsf((float)vf[ks][e]));
    const int k = dt_shift<D>(wave_max_of(bp.domax + ((int64_t)b * p.Hq + hk * p.group) * nqb, p.group * nqb), pair_max(m));
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
    const bool in = t < nqb;
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
    float* part = bp.tab_part + (((int64_t)b * p.Hq + hk * p.group + head) * bp.k_tiles + tile) * n_dist;
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
  auto issue = [&](const Step& s, lds_byte* qd, lds_byte* dd) {
    const int h = hk * p.group + s.head, valid = min(p.Sq - s.t * kBlock, kBlock);
    if (docs) next_id = doc_at(p.docs_q, (int64_t)b * p.Sq + s.t * kBlock + lane, lane < valid, -1);
    next_st = bp.stats[((int64_t)b * p.Hq + h) * (64 * nqb) + s.t * kBlock + lane];
    TL::issue(rows_rsrc<D>(p.q + b * p.qs[0] + h * p.qs[1], p.qs[2], (int64_t)s.t * kBlock, valid), q_off, wave, qd);
    TL::issue(rows_rsrc<D>(bp.dout + b * bp.dos[0] + h * bp.dos[1], bp.dos[2], (int64_t)s.t * kBlock, valid), d_off, wave, dd);
  };
  auto step = [&](const Step cur, const Step nxt, lds_byte* qt, lds_byte* dt_, lds_byte* qn, lds_byte* dn) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    const int cur_id = next_id;
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
    if (p.bias_kind == kBiasSlopes) slope = p.slopes[hk * p.group + cur.head] * kLog2e;
    __syncthreads();
    if (nxt.t >= 0) issue(nxt, qn, dn);
    if (!cur.mine) return;
    st_lse[wave][lane] = cur_st[0];
    st_del[wave][lane] = cur_st[1];
    if (docs && !cur.full) doc_ids[wave][lane] = cur_id;
    __builtin_amdgcn_wave_barrier();
    const float mul = p.k1 != 0.f ? 1.f : p.c;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int pos0 = first + cur.t * kBlock + 32 * mt + 4 * g;    // position of the lane's score 0; score r: + key_off(r)
      floatx16 s = product32<D, BF>(qt + 32 * mt * (2 * D), rd, kf), w;
      floatx16 dp = product32<D, BF>(dt_ + 32 * mt * (2 * D), rd, vf);
      if (p.k1 != 0.f) cap_scores_grad(p, s, w);
      if constexpr (TAB) {
        const int x = min(max(j - pos0, -p.radius), p.radius + kTabPad);   // distance j - p falls with the row
        const float* t = tab + (x + p.radius + kTabPad);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], mul, t[-key_off(r)]);
      } else if (p.bias_kind == kBiasSlopes) {
        const float x = (float)(j - pos0);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], mul, -slope * __builtin_fabsf(x - (float)key_off(r)));
      }
      if (!cur.full) {
        const int rel = from - pos0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = key_off(r) >= rel ? s[r] : -INFINITY;
        if (docs) doc_scores(L, &doc_ids[wave][32 * mt + 4 * g], s);
      }
      half8_t x[2];
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const floatx4 ls = *reinterpret_cast<const floatx4*>(&st_lse[wave][32 * mt + 8 * q4 + 4 * g]);
        const floatx4 de = *reinterpret_cast<const floatx4*>(&st_del[wave][32 * mt + 8 * q4 + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * q4 + e;
          const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.cc, (BF ? 0.f : (float)kPShift) - ls[e]));
          x[r >> 3][r & 7] = to_elem<BF>(pr);
          s[r] = pr * (dp[r] - de[e]);
        }
      }
      accumulate32<D, BF>(dv, dt_ + 32 * mt * (2 * D), tr, x);
      if constexpr (TAB) {
        const int d_lo = key0 - (pos0 - 4 * g) - 31, d_hi = d_lo + 62;   // distances of the piece
        if (d_lo >= p.radius || d_hi <= -p.radius) {
          float t = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) t += s[r];
          if (d_lo >= p.radius) far_hi += t; else far_lo += t;
        } else {
          float* sk = skew[wave];                 // [query][key]
#pragma unroll
          for (int r = 0; r < 16; ++r) sk[(key_off(r) + 4 * g) * 33 + j32] = s[r];
          __builtin_amdgcn_wave_barrier();
          const int dg = lane - 31;               // lane l sums the diagonal key - query = l - 31 of the piece
          float t = 0.f;
#pragma unroll 8
          for (int y = 0; y < 32; ++y) {
            const int key = y + dg;
            const bool in = key >= 0 && key < 32;
            const float e = sk[y * 33 + (in ? key : 0)];
            t += in ? e : 0.f;
          }
          __builtin_amdgcn_wave_barrier();
          if (lane < 63) {
            const int d = d_lo + lane;
            if (d >= p.radius) far_hi += t;
            else if (d <= -p.radius) far_lo += t;
            else sums[d + p.radius] += t;
          }
        }
      }
      if (p.k1 != 0.f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= w[r];
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r >> 3][r & 7] = to_elem<BF>(BF ? s[r] : s[r] * up);
      accumulate32<D, BF>(dk, qt + 32 * mt * (2 * D), tr, x);
    }
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
  const int64_t at = ((int64_t)bk * p.Sk + key0) * D;
  store_rows<D, BF>(dk, down, stage, bp.dk + at, keys, lane);
  store_rows<D, BF>(dv, BF ? 1.f : pow2(-kPShift), stage, bp.dv + at, keys, lane);
}

// ---- host side

struct Layout { int64_t stats, domax, vmax, part, total; };

Layout layout(int B, int Hq, int Hkv, int Sq, int Sk, int radius, int docs) {
  const int64_t nq = (Sq + 63) / 64, nk = (Sk + 63) / 64, kt = (Sk + 127) / 128;
  auto up = [](int64_t n) { return (n + 255) & ~(int64_t)255; };
  Layout l;
  l.stats = docs ? up((int64_t)B * (nq + nk) * (int64_t)sizeof(DocRange)) : 0;
  l.domax = l.stats + up((int64_t)B * Hq * nq * 64 * 8);
  l.vmax = l.domax + up((int64_t)B * Hq * nq * 4);
  l.part = l.vmax + up((int64_t)B * Hkv * nk * 4);
  l.total = l.part + (radius >= 0 ? up((int64_t)B * Hq * kt * (2 * radius + 1) * 4) : 0);
  return l;
}

template <int D, bool BF>
void launch_bwd(BwdParams& p, hipStream_t st) {
  const ScoreParams& s = p.s;
  const int nq = (s.Sq + 63) / 64, nk = (s.Sk + 63) / 64;
  const int n_tab = s.bias_kind == kBiasTable ? 2 * s.radius + 1 + 2 * kTabPad : 0;
  score_attn_bwd_prep_kernel<D, BF><<<dim3((unsigned)(s.B * s.Hq * nq + (BF ? 0 : s.B * s.Hkv * nk))), dim3(256), 0, st>>>(p);
  const unsigned gq = 8u * (unsigned)p.q_chunk, gk = 8u * (unsigned)p.k_chunk;
  score_attn_bwd_q_kernel<D, BF><<<dim3(gq), dim3(256), (size_t)n_tab * 4, st>>>(p);
  if (n_tab) {
    score_attn_bwd_k_kernel<D, BF, true><<<dim3(gk), dim3(256), (size_t)(n_tab + 4 * (2 * s.radius + 1)) * 4, st>>>(p);
    score_attn_bwd_table_kernel<BF><<<dim3((unsigned)((2 * s.radius + 64) / 64), (unsigned)s.Hq), dim3(256), 0, st>>>(p);
  } else {
    score_attn_bwd_k_kernel<D, BF, false><<<dim3(gk), dim3(256), 0, st>>>(p);
  }
}

}  // namespace

extern "C" int64_t stof_score_attn_bwd_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Sk, int D, int radius, int docs) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sk <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
  return layout(B, Hq, Hkv, Sq, Sk, radius, docs).total;
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
  const Layout l = layout(B, Hq, Hkv, Sq, Sk, table ? radius : -1, docs_q != nullptr);
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
  p.q_chunk = (B * Hq * p.q_tiles + 7) / 8; p.k_chunk = (B * Hkv * p.k_tiles + 7) / 8;
  hipStream_t st = (hipStream_t)stream;
  if (docs_q) score_attn_ranges(p.s, ws, st);
  if (D == 64) { if (dtype == STOF_DTYPE_BF16) launch_bwd<64, true>(p, st); else launch_bwd<64, false>(p, st); }
  else { if (dtype == STOF_DTYPE_BF16) launch_bwd<128, true>(p, st); else launch_bwd<128, false>(p, st); }
  return stof_check_launch();
}
