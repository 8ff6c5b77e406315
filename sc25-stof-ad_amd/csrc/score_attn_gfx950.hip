// Attention with score rules, forward: stof_score_attn_fwd (see score_attn.h for the rule).
//
// Two forms, the same wave program: a wave keeps 32 query rows in registers, scores are produced
// transposed (S^T = K Q^T, v_mfma_f32_32x32x16), so a lane owns ONE query: its position, limit,
// document, running maximum and sum are per-lane scalars and the rule is a register loop; P never
// touches LDS (the accumulator layout of S^T is the B operand layout of O^T = V^T P^T) and V is
// transposed by the LDS read.
//
//  * wide form: four waves x 32 queries of one head share K and V tiles of 64 keys, direct-to-LDS
//    loads double buffered, one barrier per tile.  Which tiles a workgroup visits and which of them
//    need the element test is decided for 64 tiles at a time, one tile per lane: limits and document
//    ranges become three 64-bit sets that the walk takes bit by bit.  On small grids two such sets of four waves
//    walk every other tile each (parts) and join their rows through LDS.
//  * row form, for few rows and long keys (single tokens) and for small grids: one workgroup owns 32
//    rows, row r = (query r / G, head r % G of the G heads that share a key head), so a token's heads
//    read the cache once; its eight waves take every eighth tile of 32 keys through a buffer of their own
//    without barriers, and the keys can be split further over workgroups, joined by a second kernel.
#include "score_attn.h"

namespace {

constexpr float kLazy = 8.0f;       // log2 slack before the running maximum is raised
// fp16: P is carried times 2^7, in its product and in the running sum alike.  With the slack it stays below 2^15, and a P is off
// by at most 2^-32 of the maximum's: held plainly, what lies below 2^-25 of it vanished from the product and stayed in the
// sum (65536 keys at 2^-25.2 of one other: outputs of 0 for 1.6e-3).  bfloat16 has the exponents of fp32.
template <bool BF> constexpr float kPUp = BF ? 0.f : 7.f;

// Document ranges of the 64-position blocks of both sequences: one wave per block.
__global__ __launch_bounds__(64) void doc_ranges_kernel(const ScoreParams p) { write_doc_range(p, blockIdx.x, threadIdx.x); }

// Online softmax of one wave over 16 MT scores per lane: raises the running maximum (rescaling O when it
// moves by more than kLazy), turns scores into probabilities in the tensors' format (the B operand of the
// second product) and adds to the running sum.  The sum is taken in fp32 from the unrounded
// probabilities; their rounding to 16 bits is the only one between the scores and the output.
template <int D, int MT, bool BF>
struct Softmax {
  floatx16 o[D / 32];
  float m = -INFINITY, mc = 0.f, raise_at = -INFINITY, l = 0.f;
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  }
  __device__ __forceinline__ void step(float cc, float add, const floatx16 (&s)[MT], half8_t (&pf)[MT][2]) {   // scores times cc plus add: log2 units
    float mx = s[0][0];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
    mx = __builtin_fmaf(pair_max(mx), cc, add);
    if (__any(mx > raise_at)) {
      const float m_new = mx > raise_at ? mx : m;
      const float m_sub = m_new == -INFINITY ? 0.f : m_new;   // a row that has seen no key: exp2(-inf) = 0 and no inf - inf
      const float alpha = __builtin_amdgcn_exp2f(m - m_sub);
      mc = m_sub;
      m = m_new;
      raise_at = m_new + kLazy;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
    }
    const float base = (add - mc) + kPUp<BF>;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r], cc, base));
        sum[r & 1] += e;
        pf[mt][r >> 3][r & 7] = to_elem<BF>(e);
      }
    l += sum[0] + sum[1];
  }
  // O^T += V^T P^T over the tile's 32 MT keys
  __device__ __forceinline__ void accumulate(const lds_byte* vt, const int (&tr)[D / 32][2], const half8_t (&pf)[MT][2]) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const lds_byte* vp = vt + (32 * mt + 16 * s2) * (2 * D);
          o[dt] = mfma32<BF>(lds_frag_tr(vp + tr[dt][0], vp + tr[dt][1]), pf[mt][s2], o[dt]);
        }
  }
};

// S^T = K Q^T for 32 MT keys
template <int D, int MT, bool BF>
__device__ __forceinline__ void scores_product(const lds_byte* kt, const int (&rd)[D / 16], const half8_t (&qf)[D / 16], floatx16 (&s)[MT]) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[mt][r] = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) s[mt] = mfma32<BF>(lds_frag(kt + 32 * mt * (2 * D) + rd[ks]), qf[ks], s[mt]);
}

// One row's 32-bit outputs (O^T layout: o[dt][r] of lane (j32, g) is row j32, column 32 dt + 8 (r / 4) + 4 g + r % 4)
// through the wave's LDS stage (rows of 2 D bytes, 16-byte chunks XOR-ed by the row) to memory, whole rows at a time.
template <int D, bool BF>
__device__ __forceinline__ void stage_rows(const floatx16 (&o)[D / 32], float inv, lds_byte* stage, int j32, int g) {
  constexpr int kC = D / 8 - 1;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      half4_t o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) o4[e] = to_elem<BF>(o[dt][4 * q4 + e] * inv);
      *reinterpret_cast<__attribute__((address_space(3))) half4_t*>(stage + j32 * (2 * D) + (((4 * dt + q4) ^ (j32 & kC)) << 4) + 8 * g) = o4;
    }
}

// ---- wide form.  Bound: the present order of vector issue and MFMAs.  A wave's 32 x 64 scores cost 4 D / 16 MFMAs of 32 cycles and,
// without a rule, 107 vector instructions of 4 cycles and 32 exponentials (+ 64 for slopes, 32 and as many LDS reads for a table within its
// radius, 32 and 64 transcendental for a cap).  A wave does them one after the other - all score MFMAs, the rule and the exponentials, all
// MFMAs of the second product - so that the two kinds of issue overlap only where another wave of the SIMD is in the other kind: by
// about a third.  That is this schedule's figure and no limit of the machine.  bf16, B2 H16 S2048: D64
// 50 us (685 TFLOP/s, MFMA busy 35 %), with a table 57, capped and causal 45; D128 70 us (980 TFLOP/s, 51 %), table
// 73, capped and causal 56.  Tiles of 64 keys keep a 32-row wave within 170 registers at D64 (three workgroups per unit; held to
// four it spilled: B8 H12 S1024 with a table 41 -> 50 us) and 232 at D128 (two).
//
// CAP is a template argument: with the cap behind a run-time branch the compiler computes it speculatively for every
// tile (64 transcendental operations a lane and tile beside the 32 of the softmax).
template <int D, bool BF, bool CAP, int BIAS, int KG>
__global__ __launch_bounds__(256 * KG, 2) void score_attn_wide_kernel(const ScoreParams p) {
  typedef TileLoad<D, kBlock, 4> TL;
  __shared__ __attribute__((aligned(1024))) unsigned char k0[KG * TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char k1[KG * TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char v0[KG * TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char v1[KG * TL::kBytes];
  __shared__ int doc_ids[4 * KG][kBlock];       // per wave: the documents of the current tile's keys
  extern __shared__ float tab[];                // distance table (kBiasTable)

  const int all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all_waves & 3, part = all_waves >> 2;   // (part < KG)
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;

  Placed at;
  if (!place(blockIdx.x, p.B * p.Hq, p.group, p.tiles, p.chunk, p.cus_per_xcd, KG == 2 ? 1 : D == 64 ? 3 : 2, p.causal, p.uneven, at)) return;
  const int bh = at.head, tile = p.tiles - 1 - at.rank;
  const int b = bh / p.Hq, h = bh - b * p.Hq, hk = h / p.group;

  const Sample sample = sample_of(p, b);
  const int klen = sample.keys, first = sample.first, prefix = sample.prefix;
  const int row0 = tile * 128 + 32 * wave;               // this wave's first query
  const int rows = min(p.Sq - row0, 32);                 // (<= 0: none)
  const int i = row0 + j32;
  const bool docs = p.docs_q != nullptr;

  LaneRow L;
  L.pos = first + i;
  L.limit = row_limit(p.causal, klen, prefix, L.pos);
  L.doc = docs ? doc_at(p.docs_q, (int64_t)b * p.Sq + i, i < p.Sq, -1) : 0;
  L.slope = BIAS == kBiasSlopes ? p.slopes[h] * p.slope_mul : 0.f;
  L.tab = tab;

  // Q^T as the B operand: lane (query j32, group g) holds 8 consecutive d per step; rows past the end re-read the last
  half8_t qf[D / 16];
  {
    const half_t* src = p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)min(i, p.Sq - 1) * p.qs[2];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const half8_t*>(src + 16 * ks + 8 * g);
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

  // ---- which key tiles: lane l decides tile 64 w + l
  const int wg_rows = min(p.Sq - tile * 128, 128);
  const int wg_hi = row_limit(p.causal, klen, prefix, first + tile * 128 + wg_rows - 1);
  const int my_hi = rows > 0 ? row_limit(p.causal, klen, prefix, first + row0 + rows - 1) : 0;
  const int my_lo = rows > 0 ? row_limit(p.causal, klen, prefix, first + row0) : 0;   // every row allows the keys below this
  DocRange qa = {0, 0, 1, 0}, qb = qa;                    // documents of the workgroup's two 64-row blocks
  const int nqb = (p.Sq + kBlock - 1) / kBlock, nkb = (p.Sk + kBlock - 1) / kBlock;
  if (docs) {
    const DocRange* dr = p.dr_q + (int64_t)b * nqb + 2 * tile;
    qa = dr[0];
    qb = 2 * tile + 1 < nqb ? dr[1] : DocRange{1, 0, 0, 0};
  }
  const DocRange mine = wave < 2 ? qa : qb;
  const int n_tiles = (wg_hi + kBlock - 1) / kBlock;
  const int n_win = (n_tiles + 63) >> 6;
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
  struct Step { int more; int t; int mine; int full; };       // more: some part has a tile
  int win = 0;
  if (n_win > 0) window(0);
  auto next_tile = [&]() -> Step {
    while (set_load == 0) {
      if (++win >= n_win) return Step{0, -1, 0, 0};
      window(win);
    }
    const int bit = __builtin_ctzll(set_load);
    set_load &= set_load - 1;
    return Step{1, 64 * win + bit, (int)((set_mine >> bit) & 1), (int)((set_full >> bit) & 1)};
  };
  auto next_step = [&]() -> Step {
    Step s = next_tile();
    if constexpr (KG == 2) {
      if (s.more) {
        const Step second = next_tile();
        if (part) { s = second; s.more = 1; }
      }
    }
    return s;
  };

  Softmax<D, 2, BF> sm;
  sm.init();

  int next_valid = 0, next_id = 0;   // document of key `lane` of the tile whose loads are in flight
  auto issue = [&](int t, lds_byte* kd, lds_byte* vd) {
    const int valid = min(klen - t * kBlock, kBlock);
    // (the loaded id as it is: anything computed from it here would wait for the load)
    if (docs) next_id = p.docs_k[(int64_t)b * p.Sk + t * kBlock + min(lane, valid - 1)];
    next_valid = valid;
    TL::issue(ksrc.tile(t, valid), k_off, wave, kd);
    TL::issue(vsrc.tile(t, valid), v_off, wave, vd);
  };
  auto step = [&](const Step cur, const Step nxt, lds_byte* kt, lds_byte* vt, lds_byte* kn, lds_byte* vn) {
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's share of the tile landed
    const int cur_id = lane < next_valid ? doc_or(next_id, -2) : -2;
    if (docs) {
      // keys of no document: whatever their values are, zeros take their place (0 times NaN is NaN)
      const uint64_t valid = __ballot(cur_id >= 0);
      if (~valid) TL::keep(valid, wave, lane, vt);
    }
    __syncthreads();
    if (nxt.t >= 0) issue(nxt.t, kn, vn);
    if (!cur.mine) return;
    // fragments two ahead of their MFMA, in a ring of three: K's for the scores, then V's (transposed), the first two of
    // which arrive during the softmax
    constexpr int NS = D / 8, NV = D / 8;          // MFMAs of the scores and of P V
    half8_t ring[3];
    auto fetch = [&](int n) {
      if (n < NS) {
        ring[n % 3] = lds_frag(kt + 32 * (n & 1) * (2 * D) + rd[n >> 1]);
      } else if (n < NS + NV) {
        const int m = n - NS, dt = m % (D / 32);
        const lds_byte* vp = vt + 16 * (m / (D / 32)) * (2 * D);
        ring[n % 3] = lds_frag_tr(vp + tr[dt][0], vp + tr[dt][1]);
      }
    };
    floatx16 s[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
    fetch(0);
    fetch(1);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      fetch(n + 2);
      __builtin_amdgcn_sched_barrier(0);
      s[n & 1] = mfma32<BF>(ring[n % 3], qf[n >> 1], s[n & 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const int j0 = cur.t * kBlock + 4 * g;
    if constexpr (CAP) { cap_scores(p, s[0]); cap_scores(p, s[1]); }
    float cc = p.cc, add = 0.f;
    bool look_up = true;
    if constexpr (BIAS == kBiasTable) {
      const int at = cur.t * kBlock - (first + row0);
      const FarPiece f = far_piece(p, tab, at - 31, at + kBlock - 1);
      if (f.far) { look_up = false; cc = p.c; add = f.add; }
    }
    if (look_up) {
      bias_scores<BIAS>(p, L, j0, s[0]);
      bias_scores<BIAS>(p, L, j0 + 32, s[1]);
    }
    if (!cur.full) {
      limit_scores(L, j0, s[0]);
      limit_scores(L, j0 + 32, s[1]);
      if (docs) {
        doc_ids[all_waves][lane] = cur_id;
        __builtin_amdgcn_wave_barrier();
        doc_scores(L, &doc_ids[all_waves][4 * g], s[0]);
        doc_scores(L, &doc_ids[all_waves][32 + 4 * g], s[1]);
      }
    }
    half8_t pf[2][2];
    sm.step(cc, add, s, pf);
#pragma unroll
    for (int n = NS; n < NS + NV; ++n) {
      const int m = n - NS, u = m / (D / 32), dt = m % (D / 32);
      fetch(n + 2);
      __builtin_amdgcn_sched_barrier(0);
      sm.o[dt] = mfma32<BF>(ring[n % 3], pf[u >> 1][u & 1], sm.o[dt]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  lds_byte* const ka = (lds_byte*)k0 + part * TL::kBytes;
  lds_byte* const kb = (lds_byte*)k1 + part * TL::kBytes;
  lds_byte* const va = (lds_byte*)v0 + part * TL::kBytes;
  lds_byte* const vb = (lds_byte*)v1 + part * TL::kBytes;
  Step cur = next_step();
  if (cur.t >= 0) issue(cur.t, ka, va);
  // (behind the first tile's loads, whose latency it shares; the walk's first barrier covers it)
  if constexpr (BIAS == kBiasTable) load_table<BF>(p, h, tab, threadIdx.x, 256 * KG);
  while (cur.more) {
    Step nxt = next_step();
    step(cur, nxt, ka, va, kb, vb);
    cur = nxt;
    if (nxt.more) {
      cur = next_step();
      step(nxt, cur, kb, vb, ka, va);
    }
  }

  __syncthreads();             // every wave has left the walk: the tile buffers become output stages
  lds_byte* stage = (lds_byte*)(wave == 0 ? k0 : wave == 1 ? k1 : wave == 2 ? v0 : v1);
  if constexpr (KG == 2) {
    // the second part's rows to the first: O through the second part's tile buffers, maxima and sums where the documents were
    float* od = reinterpret_cast<float*>((unsigned char*)(wave == 0 ? k0 : wave == 1 ? k1 : wave == 2 ? v0 : v1) + TL::kBytes);
    if (part) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) od[(16 * dt + r) * 64 + lane] = sm.o[dt][r];
      doc_ids[wave][lane] = __builtin_bit_cast(int, sm.m);
      doc_ids[4 + wave][lane] = __builtin_bit_cast(int, sm.l);
    }
    __syncthreads();
    if (part) return;
    const float m1 = __builtin_bit_cast(float, doc_ids[wave][lane]), l1 = __builtin_bit_cast(float, doc_ids[4 + wave][lane]);
    const float m = fmaxf(sm.m, m1);
    // a part that saw no key has the maximum -inf; one that saw only NaN too, and a sum of NaN, which must stay (a lane's sum
    // is that of its own keys: 0 where those are masked, whatever the row's maximum)
    const float e0 = __builtin_amdgcn_exp2f(sm.m - m), e1 = __builtin_amdgcn_exp2f(m1 - m);
    const float f0 = sm.m == -INFINITY ? 0.f : e0, f1 = m1 == -INFINITY ? 0.f : e1;
    sm.l = (sm.l == 0.f ? 0.f : sm.l * e0) + (l1 == 0.f ? 0.f : l1 * e1);
    sm.m = m;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) sm.o[dt][r] = sm.o[dt][r] * f0 + od[(16 * dt + r) * 64 + lane] * f1;
  }
  if (rows <= 0) return;
  const float l = pair_sum(sm.l);
  const float inv = l == 0.f ? 0.f : 1.f / l;              // no allowed key at all: zeros
  if (p.lse && g == 0 && i < p.Sq) p.lse[(int64_t)bh * p.Sq + i] = l == 0.f ? -INFINITY : (sm.m + (__builtin_amdgcn_logf(l) - kPUp<BF>) + p.lse_add) * kLn2;
  stage_rows<D, BF>(sm.o, inv, stage, j32, g);
  half_t* ob = p.out + b * p.os[0] + h * p.os[1] + (int64_t)row0 * p.os[2];
  const __amdgpu_buffer_rsrc_t o_rsrc = stof_wave_rsrc(ob);
  constexpr int kC = D / 8;
#pragma unroll
  for (int n = 0; n < 32 * kC / 64; ++n) {
    const int t = (64 / kC) * n + lane / kC, c = lane % kC;
    const half8_t o = lds_frag(stage + t * (2 * D) + ((c ^ (t & (kC - 1))) << 4));
    if (t < rows) stof_store16_through(o_rsrc, (uint32_t)t * (uint32_t)(p.os[2] * 2) + 16 * c, o);
  }
}

// ---- row form.  Grid: B * Hkv * tiles (32 rows each) * splits.
//
// Bound: the reading of K and V, or for short caches the chain of dependent loads.  Each wave keeps one K and one V
// tile of 32 keys: the next K tile is requested as soon as the scores of the current one are formed, the next V
// tile after the second product, so one of the two is always on its way while the wave computes, and
// eight waves with 128 KB of requests (head size 128) per compute unit cover the memory's latency.  One token of
// B1 H32/8 over 16384 keys, D128: 14.0 us + 4.6 us for the join (67 MB: 4.8 TB/s); B1 H12 over 512 keys 7 us.
constexpr int kRowKeys = 32;
constexpr int kRowWaves = 8;

template <int D, bool BF, bool CAP, int BIAS>
__global__ __launch_bounds__(64 * kRowWaves, 1) void score_attn_rows_kernel(const ScoreParams p) {
  typedef TileLoad<D, kRowKeys, 1> TL;
  __shared__ __attribute__((aligned(1024))) unsigned char k_lds[kRowWaves * TL::kBytes];
  __shared__ __attribute__((aligned(1024))) unsigned char v_lds[kRowWaves * TL::kBytes];
  __shared__ int doc_ids[kRowWaves][kRowKeys];
  __shared__ float stats[kRowWaves][2][64];
  extern __shared__ float tab[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;
  const int G = p.group, n_rows = p.Sq * G;

  const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
  const int tile = p.tiles - 1 - rest % p.tiles, bk = rest / p.tiles;
  const int b = bk / p.Hkv, hk = bk - b * p.Hkv;
  const Sample sample = sample_of(p, b);
  const int klen = sample.keys, first = sample.first, prefix = sample.prefix;
  const int r0 = tile * 32, rows = min(n_rows - r0, 32);
  const int r = min(r0 + j32, n_rows - 1), i = r / G, hg = r - i * G, h = hk * G + hg;
  const int i_lo = r0 / G, i_hi = (r0 + rows - 1) / G;
  const bool docs = p.docs_q != nullptr;

  // distance table of the heads in this tile: all G of them, or the rows' own when a tile has fewer rows
  const int n_tab = 2 * p.radius + 1 + 2 * kTabPad;
  LaneRow L;
  L.pos = first + i;
  L.limit = row_limit(p.causal, klen, prefix, L.pos);
  L.doc = docs ? doc_at(p.docs_q, (int64_t)b * p.Sq + i, true, -1) : 0;
  L.slope = BIAS == kBiasSlopes ? p.slopes[h] * p.slope_mul : 0.f;
  L.tab = tab + hg * n_tab;
  L.gtab = p.table + (int64_t)h * (2 * p.radius + 1);
  half8_t qf[D / 16];
  {
    const half_t* src = p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)i * p.qs[2];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *reinterpret_cast<const half8_t*>(src + 16 * ks + 8 * g);
  }
  TileSource<D, kRowKeys> ksrc, vsrc;
  ksrc.set(p.k + b * p.ks[0] + hk * p.ks[1], p.ks[2]);
  vsrc.set(p.v + b * p.vs[0] + hk * p.vs[1], p.vs[2]);
  uint32_t k_off[TL::kN], v_off[TL::kN];
  TL::offsets(k_off, 0, lane, p.ks[2]);
  TL::offsets(v_off, 0, lane, p.vs[2]);
  int rd[D / 16], tr[D / 32][2];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) rd[ks] = frag_off<D>(j32, g, ks);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) tr[dt][hh] = tr_off<D>(lane, dt, hh);

  // this wave's stream of tiles: stream + n * streams; lane l decides the (64 w + l)-th of them
  const int streams = kRowWaves * p.splits, stream = kRowWaves * split + wave;
  const int hi = row_limit(p.causal, klen, prefix, first + i_hi), lo = row_limit(p.causal, klen, prefix, first + i_lo);
  const int nqb = (p.Sq + kBlock - 1) / kBlock, nkb = (p.Sk + kBlock - 1) / kBlock;
  DocRange qa = {0, 0, 1, 0}, qb = qa;                    // the at most two blocks that hold these queries
  if (docs) {
    qa = p.dr_q[(int64_t)b * nqb + i_lo / kBlock];
    qb = p.dr_q[(int64_t)b * nqb + i_hi / kBlock];
  }
  const int n_tiles = (hi + kRowKeys - 1) / kRowKeys;
  const int n_mine = stream < n_tiles ? (n_tiles - stream + streams - 1) / streams : 0;
  const int n_win = (n_mine + 63) >> 6;
  uint64_t set_load = 0, set_full = 0;
  auto window = [&](int w) {
    const int n = 64 * w + lane, t = stream + n * streams, j0 = t * kRowKeys;
    bool load = n < n_mine, full = j0 + kRowKeys <= lo;
    if (docs && load) {
      const DocRange rk = p.dr_k[(int64_t)b * nkb + j0 / kBlock];
      load = ranges_meet(rk, qa) || ranges_meet(rk, qb);
      full = full && ranges_one(rk, qa) && ranges_one(rk, qb);
    }
    set_load = __ballot(load); set_full = __ballot(full);
  };
  struct Step { int t; int full; };
  int win = 0;
  if (n_win > 0) window(0);
  auto next_step = [&]() -> Step {
    while (set_load == 0) {
      if (++win >= n_win) return Step{-1, 0};
      window(win);
    }
    const int bit = __builtin_ctzll(set_load);
    set_load &= set_load - 1;
    return Step{stream + (64 * win + bit) * streams, (int)((set_full >> bit) & 1)};
  };

  Softmax<D, 1, BF> sm;
  sm.init();
  lds_byte* kt = (lds_byte*)k_lds + wave * TL::kBytes;
  lds_byte* vt = (lds_byte*)v_lds + wave * TL::kBytes;
  auto issue_k = [&](int t) { TL::issue(ksrc.tile(t, min(klen - t * kRowKeys, kRowKeys)), k_off, 0, kt); };
  auto issue_v = [&](int t) { TL::issue(vsrc.tile(t, min(klen - t * kRowKeys, kRowKeys)), v_off, 0, vt); };
  // every LDS read so far has returned, so loads may overwrite what was read
  auto drained = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    asm volatile("" ::: "memory");
  };
  constexpr int kAllButOne = (TL::kN & 15) | ((TL::kN >> 4) << 14) | 0x0F70;   // vmcnt: the loads of one tile may be out
  Step cur = next_step();
  if (cur.t >= 0) { issue_k(cur.t); issue_v(cur.t); }
  if (BIAS == kBiasTable && p.table_in_lds) {      // (behind the first loads, whose latency it shares)
    for (int x = 0; x < G; ++x) load_table<BF>(p, hk * G + x, tab + x * n_tab, threadIdx.x, 64 * kRowWaves);
    __syncthreads();
  }
  while (cur.t >= 0) {
    const Step nxt = next_step();
    int id = 0;
    if (docs) {
      const int jj = cur.t * kRowKeys + j32;
      id = doc_at(p.docs_k, (int64_t)b * p.Sk + jj, jj < klen, -2);     // (its wait covers both tiles)
      doc_ids[wave][j32] = id;
      __builtin_amdgcn_wave_barrier();
    }
    __builtin_amdgcn_s_waitcnt(kAllButOne);       // K has landed (V, requested after it, may be out)
    asm volatile("" ::: "memory");
    floatx16 s[1];
    scores_product<D, 1, BF>(kt, rd, qf, s);
    drained();
    if (nxt.t >= 0) issue_k(nxt.t);
    const int j0 = cur.t * kRowKeys + 4 * g;
    if constexpr (CAP) cap_scores(p, s[0]);
    if (BIAS == kBiasTable && !p.table_in_lds) {
      // more heads share the cache than tables fit: entries straight from memory
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int x = min(max(j0 + key_off(r) - L.pos, -p.radius), p.radius) + p.radius;
        s[0][r] = __builtin_fmaf(s[0][r], p.c, table_entry<BF>(L.gtab[x]));
      }
    } else {
      bias_scores<BIAS>(p, L, j0, s[0]);
    }
    if (!cur.full) {
      limit_scores(L, j0, s[0]);
      if (docs) doc_scores(L, &doc_ids[wave][4 * g], s[0]);
    }
    half8_t pf[1][2];
    sm.step(p.cc, 0.f, s, pf);
    if (nxt.t >= 0) __builtin_amdgcn_s_waitcnt(kAllButOne);             // V has landed (the next K may be out)
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("" ::: "memory");
    if (docs) {
      const uint64_t valid = __ballot(id >= 0);
      if (~valid) TL::keep(valid, 0, lane, vt);
    }
    sm.accumulate(vt, tr, pf);
    drained();
    if (nxt.t >= 0) issue_v(nxt.t);
    cur = nxt;
  }

  // ---- join the waves: maxima and sums through `stats`, O (32 x D floats a wave) through the tile buffers
  // (a wave's K and V tiles hold just that: registers below D / 4 in the K tiles, the rest in the V tiles), a
  // share of the columns joined by each wave
  stats[wave][0][lane] = sm.m;
  stats[wave][1][lane] = sm.l;
  __syncthreads();             // (also: every wave has left the walk)
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) m = fmaxf(m, stats[w][0][lane]);
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    // (a wave that saw no key has the sum 0; one that saw only NaN has the maximum -inf too, and the sum NaN, which must stay)
    const float lw = stats[w][1][lane];
    l += lw == 0.f ? 0.f : lw * __builtin_amdgcn_exp2f(stats[w][0][lane] - m);
  }
  const float f = sm.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm.m - m);
  constexpr int kRegs = D / 2;                          // registers of O: index 16 dt + x
  constexpr int kHalf = kRegs / 2;
  float* klo = reinterpret_cast<float*>(k_lds);
  float* vhi = reinterpret_cast<float*>(v_lds);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int n = 16 * dt + x;
      (n < kHalf ? klo : vhi)[wave * (TL::kBytes / 4) + (n % kHalf) * 64 + lane] = sm.o[dt][x] * f;
    }
  __syncthreads();
  l = pair_sum(l);
  constexpr int kPer = kRegs / kRowWaves;               // register indices per wave
  float part[kPer];
  const float* from = (kPer * wave < kHalf ? klo : vhi) + (kPer * wave % kHalf) * 64 + lane;
#pragma unroll
  for (int x = 0; x < kPer; ++x) {
    part[x] = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) part[x] += from[w * (TL::kBytes / 4) + x * 64];
  }
  // register index n = kPer * wave + x of lane (j32, g): row j32, column 32 (n / 16) + 8 ((n % 16) / 4) + 4 g + n % 4
  if (j32 >= rows) return;
  if (p.splits > 1) {
    const int64_t slot = ((int64_t)bk * p.tiles + tile) * p.splits + split;
    float* po = p.part + slot * (32 * D + 64) + j32 * D;
#pragma unroll
    for (int x = 0; x < kPer; x += 4) {
      const int n = kPer * wave + x, col = 32 * (n / 16) + 8 * ((n % 16) / 4) + 4 * g;
      *reinterpret_cast<floatx4*>(po + col) = floatx4{part[x], part[x + 1], part[x + 2], part[x + 3]};
    }
    if (wave == 0 && g == 0) {
      float* ps = p.part + slot * (32 * D + 64) + 32 * D;
      ps[j32] = m;
      ps[32 + j32] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  half_t* orow = p.out + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
#pragma unroll
  for (int x = 0; x < kPer; x += 4) {
    const int n = kPer * wave + x, col = 32 * (n / 16) + 8 * ((n % 16) / 4) + 4 * g;
    half4_t o4;
#pragma unroll
    for (int e = 0; e < 4; ++e) o4[e] = to_elem<BF>(part[x + e] * inv);
    *reinterpret_cast<half4_t*>(orow + col) = o4;
  }
  if (p.lse && wave == 0 && g == 0) p.lse[((int64_t)b * p.Hq + h) * p.Sq + i] = l == 0.f ? -INFINITY : (m + (__builtin_amdgcn_logf(l) - kPUp<BF>) + p.lse_add) * kLn2;
}

// Joins the splits of the row form: one workgroup per row, every fourth split to a wave, D / 64 columns per lane; the
// waves' sums are added in their order.
template <int D, bool BF>
__global__ __launch_bounds__(256) void score_attn_join_kernel(const ScoreParams p) {
  constexpr int kC = D / 64, kSlot = 32 * D + 64;
  __shared__ float sums[4][D];
  __shared__ float factor[64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n_rows = p.Sq * p.group;
  const int64_t bk = blockIdx.x / n_rows;
  const int r = blockIdx.x - (int)bk * n_rows, tile = r / 32, j = r % 32;
  const float* base = p.part + (bk * p.tiles + tile) * p.splits * kSlot;
  // lane s: maximum and sum of split s (at most 64)
  const float ms = lane < p.splits ? base[lane * kSlot + 32 * D + j] : -INFINITY;
  const float ls = lane < p.splits ? base[lane * kSlot + 32 * D + 32 + j] : 0.f;
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float fs = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
  const float l = wave_sum(fs * ls);
  factor[lane] = fs;                                    // (every wave the same)
  __syncthreads();
  float o[kC] = {};
#pragma unroll 4
  for (int s = wave; s < p.splits; s += 4) {
    const float f = factor[s];
#pragma unroll
    for (int x = 0; x < kC; ++x) {
      const float v = base[s * kSlot + j * D + kC * lane + x];
      o[x] += f == 0.f ? 0.f : f * v;                   // (a split that saw no key, or only NaN: then l is NaN)
    }
  }
#pragma unroll
  for (int x = 0; x < kC; ++x) sums[wave][kC * lane + x] = o[x];
  __syncthreads();
  if (wave != 0) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int b = (int)(bk / p.Hkv), hk = (int)(bk - (int64_t)b * p.Hkv), i = r / p.group, h = hk * p.group + r % p.group;
  half_t* orow = p.out + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
#pragma unroll
  for (int x = 0; x < kC; ++x) {
    const int c = kC * lane + x;
    orow[c] = to_elem<BF>(((sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c])) * inv);
  }
  if (p.lse && lane == 0) p.lse[((int64_t)b * p.Hq + h) * p.Sq + i] = l == 0.f ? -INFINITY : (m + (__builtin_amdgcn_logf(l) - kPUp<BF>) + p.lse_add) * kLn2;
}

}  // namespace

// ---- host side

// Form, parts and number of key splits (us at 16 bits, D64 unless said otherwise).
//  * The row form takes calls whose rows fit one 32-row tile per key head (single tokens: a token's heads read the cache
//    once) and grids whose row tiles are all on the device at once, where a workgroup of the wide form would walk
//    all keys alone.  Wide form in two parts | row form: B1 H12 S512 9.9 | 8.7, B1 H8 S1024 14.9 | 9.3, D128 19.8 | 16.0;
//    with more row tiles than units B1 H20 queries 512 keys 1024 15.0 | 16.0, B2 H12 S512 10.3 | 11.3, D128 13.3 | 19.4.
//  * The wide form walks the keys in two parts while every workgroup can have a compute unit to itself: 256
//    workgroups, B2 H8 S2048, one part | two: 31.8 | 28.3, causal 29.9 | 25.2, D128 causal 42.1 | 35.0; 384, B8 H12 S512
//    13.9 | 17.9, B3 H8 S2048 44.7 | 50.2.
//    (256 units, as every MI355X has: the workspace's size is asked for without a device.)
//  * Splitting costs a launch (3 us) and the partial results.  Past 2048 keys the row form's splits give every unit a workgroup:
//    64 workgroups over 4096 keys 20.6 unsplit, 13.8 with four splits, 18.8 with six, over 16384 keys 64.8 | 25.2 | 35.3;
//    but 2048 keys 12.1 | 13.6 | 16.3.  Single tokens of many heads are bound by memory and gain from splits only what
//    evens out caches of different length: 128 workgroups, equal | uneven lengths, D128 over 16384 keys 203 | 179 unsplit, 186 | 129
//    with four splits, 190 | 130 with eight, over 4096 keys 41 | 32 unsplit, 47 | 34 with four.  These figures are of 64 and of 128
//    workgroups; single tokens of 65 to 127 workgroups follow the rule of 128 without a measurement of their own.
namespace {

struct Form { bool rows; int parts, tiles, splits; };

// whether the tables of the heads that share a key head fit into LDS (beside 133 KB of tiles)
inline bool tables_fit(int group, int radius) { return group * (2 * radius + 1 + 2 * kTabPad) * 4 <= 26 * 1024; }

inline Form pick_form(int B, int Hq, int Hkv, int Sq, int Sk, int form) {
  const int group = Hq / Hkv, cus = 256;
  const int64_t rows = (int64_t)Sq * group, tiles = (rows + 31) / 32, wgs = (int64_t)B * Hkv * tiles;
  const bool use_rows = form == 1 || (form < 0 && (tiles == 1 || wgs <= cus));
  if (!use_rows) {
    const int wide_tiles = (Sq + 127) / 128;
    return Form{false, form == 2 || (form < 0 && (int64_t)B * Hq * wide_tiles <= cus) ? 2 : 1, wide_tiles, 1};
  }
  int64_t splits = Sk > 2048 && wgs < cus ? cus / wgs : 1;
  if (tiles == 1 && wgs > 64 && wgs < cus) splits = Sk >= 8192 ? 4 : 1;
  const int64_t most = ((Sk + kRowKeys - 1) / kRowKeys + 2 * kRowWaves - 1) / (2 * kRowWaves);   // two tiles per wave
  if (splits > most) splits = most;
  if (splits > 64) splits = 64;                                            // one lane each in the join
  if (splits < 1) splits = 1;                                              // no keys: the outputs are still written
  return Form{true, 1, (int)tiles, (int)splits};
}

inline int64_t ranges_bytes(int B, int Sq, int Sk) {
  return (int64_t)B * ((Sq + kBlock - 1) / kBlock + (Sk + kBlock - 1) / kBlock) * (int64_t)sizeof(DocRange);
}

}  // namespace

int score_attn_check(const void* const* req, int n_req, const int64_t* const* strides, int n_strides, int B, int Hq, int Hkv, int Sq, int Sk, int D,
                     int dtype, float scale, float cap, int radius) {
  for (int i = 0; i < n_req; ++i) {
    if (!req[i]) return STOF_ERR_NULL_POINTER;
    if (!stof_aligned16(req[i])) return STOF_ERR_MISALIGNED;
  }
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sk < 0 || Hq % Hkv != 0) return STOF_ERR_BAD_SHAPE;
  if ((int64_t)B * Hq * ((Sq + 31) / 32) > 0x3fffffff || (int64_t)B * Hq * (int64_t)((Sk + 31) / 32) > 0x3fffffff || Sq > (1 << 29) || Sk > (1 << 29)) return STOF_ERR_BAD_SHAPE;
  if (D != 64 && D != 128) return STOF_ERR_UNSUPPORTED;
  if (dtype != STOF_DTYPE_F16 && dtype != STOF_DTYPE_BF16) return STOF_ERR_UNSUPPORTED;
  if (!(scale >= 1e-6f) || scale > 1e6f || !(cap >= 0.f) || cap > STOF_SCORE_MAX_CAP || (cap > 0.f && cap < 1e-3f)) return STOF_ERR_UNSUPPORTED;
  if (radius > STOF_SCORE_MAX_RADIUS) return STOF_ERR_UNSUPPORTED;
  for (int i = 0; i < n_strides; ++i) {
    if (!strides[i]) return STOF_ERR_NULL_POINTER;
    for (int j = 0; j < 3; ++j)
      if (strides[i][j] % 8 != 0 || strides[i][j] < 0) return STOF_ERR_MISALIGNED;
    if (strides[i][2] > (1 << 23)) return STOF_ERR_BAD_SHAPE;   // 64 rows of a tile stay below 2^31 bytes
  }
  return STOF_OK;
}

void score_attn_params(ScoreParams& p, const void* q, const void* k, const void* v, const void* table, const void* slopes, const void* prefix,
                       const void* kv_len, const void* docs_q, const void* docs_k, float scale, float cap, int radius, int causal, int q_start,
                       int q_end, const int64_t* qs, const int64_t* ks, const int64_t* vs, int B, int Hq, int Hkv, int Sq, int Sk) {
  p.q = (const half_t*)q; p.k = (const half_t*)k; p.v = (const half_t*)v;
  for (int j = 0; j < 3; ++j) { p.qs[j] = qs[j]; p.ks[j] = ks[j]; p.vs[j] = vs[j]; }
  p.table = (const half_t*)table; p.slopes = (const float*)slopes;
  p.prefix = (const int*)prefix; p.kv_len = (const int*)kv_len;
  p.docs_q = (const int*)docs_q; p.docs_k = (const int*)docs_k;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.group = Hq / Hkv;
  p.radius = radius < 0 ? 0 : radius;
  p.causal = causal != 0; p.q_start = q_start; p.q_end = q_end != 0;
  p.c = cap > 0.f ? 2.f * cap * kLog2e : scale * kLog2e;
  p.k1 = cap > 0.f ? 2.f * scale * kLog2e / cap : 0.f;
  p.lse_add = cap * kLog2e;
  int cus = stof_device_compute_units();
  p.cus_per_xcd = cus >= 8 ? cus / 8 : 32;
  // Samples of different work, and key heads that do not divide over the XCDs or leave each of them only some of the samples
  // (us, whole key heads | spread): lengths, B2 H16/4 S2048 D128 forward 68 | 51, backward 287 | 242, B3 H12 S2048 D64 56 | 50
  // and 215 | 147; documents, B3 H8/4 S2048 D64 41 | 35 and 109 | 94.  Twelve key heads or more that divide reach every XCD from
  // most samples, and keep their L2: lengths, B8 H12 S1024 27.7 | 29.7.  So do documents that divide (B2 H16/4
  // S2048 D128, mean of three: 32 | 33).
  const bool divides = (int64_t)B * Hkv % 8 == 0;
  const bool uneven = divides ? kv_len && Hkv < 8 : kv_len || docs_q;
  p.uneven = !uneven ? kEven : Hq % 8 == 0 ? kUnevenHeads : kUnevenTiles;
  p.cc = table ? 1.f : p.c;
  p.slope_mul = kLog2e / p.c;
}

int score_attn_ranges_at(ScoreParams& p, void* ws) {
  const int nq = (p.Sq + kBlock - 1) / kBlock, nk = (p.Sk + kBlock - 1) / kBlock;
  p.dr_q = (DocRange*)ws;
  p.dr_k = p.dr_q + (int64_t)p.B * nq;
  return p.B * (nq + nk);
}

template <int D, bool BF, bool CAP, int BIAS>
static void launch_form(ScoreParams& p, const Form& f, hipStream_t st) {
  const int n_tab = BIAS == kBiasTable ? 2 * p.radius + 1 + 2 * kTabPad : 0;
  if (f.rows) {
    const unsigned grid = (unsigned)(p.B * p.Hkv) * (unsigned)p.tiles * (unsigned)p.splits;
    score_attn_rows_kernel<D, BF, CAP, BIAS><<<dim3(grid), dim3(64 * kRowWaves), (size_t)(p.table_in_lds ? p.group * n_tab : 0) * 4, st>>>(p);
  } else {
    p.chunk = (p.B * p.Hq * p.tiles + 7) / 8;
    const dim3 grid(8u * (unsigned)p.chunk);
    if (f.parts == 2) score_attn_wide_kernel<D, BF, CAP, BIAS, 2><<<grid, dim3(512), (size_t)n_tab * 4, st>>>(p);
    else score_attn_wide_kernel<D, BF, CAP, BIAS, 1><<<grid, dim3(256), (size_t)n_tab * 4, st>>>(p);
  }
}
template <int D, bool BF, bool CAP>
static void launch_bias(ScoreParams& p, const Form& f, hipStream_t st) {
  if (p.table) launch_form<D, BF, CAP, kBiasTable>(p, f, st);
  else if (p.slopes) launch_form<D, BF, CAP, kBiasSlopes>(p, f, st);
  else launch_form<D, BF, CAP, kBiasNone>(p, f, st);
}
template <int D, bool BF>
static void launch_fwd(ScoreParams& p, const Form& f, hipStream_t st) {
  p.k1 != 0.f ? launch_bias<D, BF, true>(p, f, st) : launch_bias<D, BF, false>(p, f, st);
  if (p.splits > 1) {
    const int64_t n = (int64_t)p.B * p.Hkv * p.Sq * p.group;
    score_attn_join_kernel<D, BF><<<dim3((unsigned)n), dim3(256), 0, st>>>(p);
  }
}

extern "C" int64_t stof_score_attn_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Sk, int D, int docs, int form) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || Sk < 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
  const Form f = pick_form(B, Hq, Hkv, Sq, Sk, form);
  int64_t n = docs ? ranges_bytes(B, Sq, Sk) : 0;
  if (f.splits > 1) n += (int64_t)B * Hkv * f.tiles * f.splits * (32 * D + 64) * 4;
  return n;
}

extern "C" int stof_score_attn_fwd(const void* q, const void* k, const void* v, void* out, float* lse,
                                   const void* table, const float* slopes, const int32_t* prefix, const int32_t* kv_len,
                                   const int32_t* docs_q, const int32_t* docs_k,
                                   float scale, float cap, int radius, int causal, int q_start, int q_end,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* out_strides,
                                   int B, int Hq, int Hkv, int Sq, int Sk, int D, int dtype, int form,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  const void* req[] = {q, k, v, out};
  const int64_t* str[] = {q_strides, k_strides, v_strides, out_strides};
  const int rc = score_attn_check(req, 4, str, 4, B, Hq, Hkv, Sq, Sk, D, dtype, scale, cap, table ? radius : -1);
  if (rc) return rc;
  if (table && slopes) return STOF_ERR_UNSUPPORTED;
  if (table && radius < 0) return STOF_ERR_BAD_SHAPE;
  if ((docs_q == nullptr) != (docs_k == nullptr)) return STOF_ERR_NULL_POINTER;
  if (q_end && !kv_len) return STOF_ERR_NULL_POINTER;
  if (q_start > (1 << 29) || q_start < -(1 << 29)) return STOF_ERR_BAD_SHAPE;
  if (form < -1 || form > 2) return STOF_ERR_UNSUPPORTED;
  const Form f = pick_form(B, Hq, Hkv, Sq, Sk, form);
  const int64_t need = stof_score_attn_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, docs_q != nullptr, form);
  if (need > 0) {
    if (!workspace) return STOF_ERR_NULL_POINTER;
    if (!stof_aligned16(workspace)) return STOF_ERR_MISALIGNED;
    if (workspace_bytes < need) return STOF_ERR_BAD_SHAPE;
  }
  ScoreParams p = {};
  score_attn_params(p, q, k, v, table, slopes, prefix, kv_len, docs_q, docs_k, scale, cap, radius, causal, q_start, q_end,
                    q_strides, k_strides, v_strides, B, Hq, Hkv, Sq, Sk);
  p.out = (half_t*)out; p.lse = lse;
  for (int j = 0; j < 3; ++j) p.os[j] = out_strides[j];
  p.tiles = f.tiles; p.splits = f.splits;
  p.table_in_lds = table && tables_fit(p.group, radius);
  hipStream_t st = (hipStream_t)stream;
  if (docs_q) doc_ranges_kernel<<<dim3((unsigned)score_attn_ranges_at(p, workspace)), dim3(64), 0, st>>>(p);
  p.part = (float*)((char*)workspace + (docs_q ? ranges_bytes(B, Sq, Sk) : 0));
  if (D == 64) { if (dtype == STOF_DTYPE_BF16) launch_fwd<64, true>(p, f, st); else launch_fwd<64, false>(p, f, st); }
  else { if (dtype == STOF_DTYPE_BF16) launch_fwd<128, true>(p, f, st); else launch_fwd<128, false>(p, f, st); }
  return stof_check_launch();
}
