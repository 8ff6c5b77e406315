// Shared pieces of the attention kernels with score rules (score_attn_gfx950.hip: forward,
// score_attn_bwd_gfx950.hip: backward).
//
// Query i of a sample stands at position p_i = first + i, query head h reads key head
// h / (Hq / Hkv).  With c = scale * log2(e) the kernels work on scores in units of log2:
//     t_ij = c q_i.k_j                                        without a cap
//     t_ij = cap' + 2 cap' u_ij, u_ij = -1 / (1 + exp2(2 c q_i.k_j / cap'))    cap' = cap * log2(e): cap tanh(scale q.k / cap)
//     t_ij += table[h][clip(j - p_i, -R, R) + R] * log2(e)     or   t_ij -= slope_h * log2(e) * |p_i - j|
// over the allowed keys j < limit_i (and of the query's document), where limit_i = kv_len, or
// min(kv_len, max(p_i + 1, prefix)) for a causal rule: every mask but the documents is one
// per-row limit.  A row without allowed keys yields zeros, lse = -inf and no gradients.
//
// A capped score is kept as u: its constant cap' changes no probability and its factor 2 cap' goes into the
// multiply-add before the exponential, where the factor c of an uncapped score goes.  So `raw` below is q.k or u, p.c
// what turns it into log2 units, and cap' is only added to lse.
#pragma once
#include "stof_common.h"

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(3))) void lds_void;
typedef float floatx2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4_t lds_short4;

enum { kBiasNone = 0, kBiasTable = 1, kBiasSlopes = 2 };

constexpr int kBlock = 64;          // keys per tile, and rows per block of the document ranges
constexpr int kTabPad = 32;         // entries by which the table in LDS continues its two ends
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Finite table entries are held inside +-kTabMax (log2 units): the lowest value of the bfloat16
// format times log2(e) would otherwise become -inf, that is a masked key instead of a very small one.
constexpr float kTabMax = 1.0e38f;

// Smallest and largest document of a block of 64 positions over its valid (non-negative) ids, and
// whether all its ids are valid.  No valid id: lo > hi, which no range intersects.
struct DocRange { int lo, hi, all, pad; };
// Whether two blocks can hold a pair of one document, and whether all their pairs are of one document.
__device__ __forceinline__ bool ranges_meet(const DocRange& a, const DocRange& b) {
  return a.lo <= b.hi && b.lo <= a.hi && a.lo <= a.hi && b.lo <= b.hi;
}
__device__ __forceinline__ bool ranges_one(const DocRange& a, const DocRange& b) {
  return a.all && b.all && a.lo == a.hi && b.lo == b.hi && a.lo == b.lo;
}

// That of block `blk` of a sequence of S documents, by one wave; every lane gets it.
__device__ __forceinline__ DocRange doc_range(const int* docs, int S, int blk, int lane) {
  const int i = blk * kBlock + lane;
  const bool inside = i < S;
  const int d = inside ? docs[i] : -1;
  int lo = d >= 0 ? d : 0x7fffffff, hi = d >= 0 ? d : -1;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o, 64)); hi = max(hi, __shfl_xor(hi, o, 64)); }
  return DocRange{lo, hi, !__any(inside && d < 0), 0};
}

struct ScoreParams {
  const half_t* q; const half_t* k; const half_t* v; half_t* out; float* lse;
  int64_t qs[3], ks[3], vs[3], os[3];      // element strides (batch, head, row)
  const half_t* table; const float* slopes;
  const int* prefix; const int* kv_len;    // per sample, or NULL
  const int* docs_q; const int* docs_k;    // [B, Sq], [B, Sk], or NULL
  const DocRange* dr_q; const DocRange* dr_k;   // [B, ceil(Sq / 64)], [B, ceil(Sk / 64)]
  int B, Hq, Hkv, Sq, Sk;
  int radius, causal;
  int q_start, q_end;                      // p_0 = q_start, or kv_len - Sq with q_end
  int tiles, chunk, cus_per_xcd;           // workgroups per (batch, head); workgroups per XCD; compute units of an XCD
  int uneven;                              // placement of the query kernels, see place()
  float c, k1, lse_add;                    // raw scores to log2 units: scale log2e, or 2 cap log2e; 2 scale log2e / cap (0: no cap); cap log2e or 0
  float cc, slope_mul;                     // what turns a rule's result into log2 units: c when it is in raw units, else 1 (tables); slopes to raw units
  // form for few rows
  int splits, group, table_in_lds; float* part;
};

// Keys j < row_limit are allowed for a query at position `pos` (documents aside).
__device__ __forceinline__ int row_limit(int causal, int klen, int prefix, int pos) {
  return causal ? min(klen, max(pos + 1, prefix)) : klen;
}
// A sample's scalars: number of keys that any of its queries may see (those past it are never loaded), position of
// query 0, prefix.
struct Sample { int keys, first, prefix; };
__device__ __forceinline__ Sample sample_of(const ScoreParams& p, int b) {
  Sample s;
  s.keys = p.kv_len ? min(max(__builtin_amdgcn_readfirstlane(p.kv_len[b]), 0), p.Sk) : p.Sk;
  s.first = p.q_end ? s.keys - p.Sq : p.q_start;
  s.prefix = p.prefix ? __builtin_amdgcn_readfirstlane(p.prefix[b]) : 0;
  s.keys = max(row_limit(p.causal, s.keys, s.prefix, s.first + p.Sq - 1), 0);
  return s;
}

__device__ __forceinline__ float pair_max(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// Workgroup -> (head, tile).  The dispatcher hands workgroups to the 8 XCDs in turn and, inside an XCD, to its compute
// units in turn; an XCD takes whole key heads (with the `group` query heads that share each), so that a head's K and V
// pass through one L2, and every eighth of them, so that samples of uneven length spread over the XCDs (B8 H12 S1024
// with uneven key lengths: a sample per XCD before, the longest set the time).  Causal work grows along the
// tiles: the heads of a set that fills the XCD (`resident` workgroups per unit) are then ordered together, longest
// tiles first.  The passes over the units that become resident at once are dealt in boustrophedon order, so that a
// unit that starts with a long tile gets a short one beside it; what follows goes to whichever unit is free.
// rank counts tiles from the longest; the order is a bijection for any sizes.  Head by head, longest first, before:
// B2 H16 S2048 causal, D128: forward 65 -> 52 us, backward 113 -> 83 (queries) and 132 -> 97 (keys).
//
// `uneven` work (samples of different documents or lengths; the rules stand where it is set): whole key heads would leave an XCD with
// some of the samples only, so the query heads of every sample are dealt to all XCDs, or, where they do not divide, all
// tiles in turn.  The latter, longest first, is also the order of causal work whose key heads do not divide (B3 H12
// S2048 D64 causal: forward 53 -> 37 us, backward 136 -> 119).
enum { kEven = 0, kUnevenHeads = 1, kUnevenTiles = 2 };
struct Placed { int head, rank; };
__device__ __forceinline__ bool place(const int index, const int heads, int group, const int tiles, const int chunk,
                                      const int cus_per_xcd, const int resident, const bool graded, const int uneven, Placed& out) {
  const int x = index & 7, i = index >> 3;
  if (uneven == kUnevenHeads) group = 1;
  if (uneven == kUnevenTiles || (graded && (heads / group) % 8 != 0)) {     // (turned by one head per rank: 8 heads would else be 8 XCDs)
    out.rank = index / heads;
    out.head = (index - out.rank * heads + out.rank) % heads;
    return out.rank < tiles;
  }
  if ((heads / group) % 8 != 0) {          // key heads do not divide over the XCDs: contiguous shares, head by head
    const int id = x * chunk + i;
    out.head = id / tiles;
    out.rank = id - out.head * tiles;
    return id < heads * tiles;
  }
  const int hx = heads / 8;                // (the grid is exact: chunk = hx * tiles)
  int local;                               // of this XCD's heads
  if (!graded) {
    local = i / tiles;
    out.rank = i - local * tiles;
  } else {
    const int hs = min(hx, max(1, (resident * cus_per_xcd + tiles - 1) / tiles));
    const int set = i / (hs * tiles), h0 = set * hs, hn = min(hs, hx - h0), il = i - set * hs * tiles;
    const int pass = il / cus_per_xcd, pos = il - pass * cus_per_xcd;
    const int len = min(cus_per_xcd, hn * tiles - pass * cus_per_xcd);
    const int j = pass * cus_per_xcd + (pass < resident && (pass & 1) ? len - 1 - pos : pos);
    out.rank = j / hn;
    local = h0 + (j - out.rank * hn);
  }
  const int key_head = local / group;
  out.head = (key_head * 8 + x) * group + (local - key_head * group);
  return true;
}

// LDS tile: unpadded rows of D elements, the 16-byte chunk c of row r at chunk position c ^ swz(r).
// 128-byte rows: row bits 1, 2, 3 onto chunk bits 2, 0, 1 (two rows fill the 64 banks); 256-byte rows:
// row bits 0, 1 onto chunk bits 2, 3 and row bits 2, 3 onto chunk bits 0, 1.  The 16 rows of a fragment
// read then take 16 different chunks, the four rows of a transposing read four different 64-byte groups.
template <int D> __device__ __forceinline__ int swz(int row) {
  if constexpr (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else return ((row & 3) << 2) | ((row >> 2) & 3);
}

// Byte offsets inside a tile of the two fragment reads of lane (j32, g):
//  * rows as the A operand (v_mfma_f32_32x32x16: row j32, 8 elements from 16 ks + 8 g): frag_off + 32 rows * pitch;
//  * columns as the A operand through the transposing read: element row 8 hh + 4 g + (0..3), column 32 dt + j32.
template <int D> __device__ __forceinline__ int frag_off(int j32, int g, int ks) {
  return j32 * (2 * D) + (((2 * ks + g) ^ swz<D>(j32)) << 4);
}
template <int D> __device__ __forceinline__ int tr_off(int lane, int dt, int hh) {
  const int g = lane >> 5, j = lane & 15, dh = (lane >> 4) & 1;
  const int row = 8 * hh + 4 * g + (j >> 2);
  const int chunk = 4 * dt + 2 * dh + ((j >> 1) & 1);
  return row * (2 * D) + ((chunk ^ swz<D>(row)) << 4) + 8 * (j & 1);
}
__device__ __forceinline__ half8_t lds_frag(const lds_byte* p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) half8_t*>(p);
}
__device__ __forceinline__ half8_t lds_frag_tr(const lds_byte* p0, const lds_byte* p1) {
  const short4_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)p0);
  const short4_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)p1);
  return __builtin_bit_cast(half8_t, (short8_t)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A [rows, D] operand whose tiles are loaded: base address, bytes of a row and of a tile of ROWS rows.  Tile t becomes a
// buffer resource with its base in scalar registers and its extent up to the last of `valid` rows, so rows
// past it arrive as zeros whatever memory holds there.  (The 64-bit base per tile keeps operands beyond
// 2^32 bytes possible; strides are below 2^23 elements, so everything inside a tile fits 32 bits.)
template <int D, int ROWS> struct TileSource {
  uint64_t base; uint32_t row_bytes;
  __device__ __forceinline__ void set(const half_t* p, int64_t stride) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    // (through uint32_t: readfirstlane returns a signed int, whose upper half would be its sign)
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    base = ((uint64_t)hi << 32) | lo;
    row_bytes = (uint32_t)stride * 2;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(int t, int valid) const {
    const uint64_t a = base + (uint64_t)(uint32_t)t * (uint64_t)(ROWS * row_bytes);
    const uint32_t bytes = (uint32_t)(valid - 1) * row_bytes + 2 * D;
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(a), 0, (int)bytes, 0x00020000);
  }
};

// Direct-to-LDS load of a tile of ROWS rows by WAVES waves: one instruction brings 1 KB (1024 / (2 D) rows).
template <int D, int ROWS, int WAVES> struct TileLoad {
  static constexpr int kPitch = 2 * D;
  static constexpr int kRowsPI = 1024 / kPitch;
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kN = ROWS / kRowsPI / WAVES;     // instructions per wave
  static constexpr int kBytes = ROWS * kPitch;
  static __device__ __forceinline__ int row(int wave, int lane, int i) { return kRowsPI * (kN * wave + i) + lane / kChunks; }
  static __device__ __forceinline__ void offsets(uint32_t (&off)[kN], int wave, int lane, int64_t stride) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = row(wave, lane, i);
      off[i] = (uint32_t)r * (uint32_t)(stride * 2) + 16 * ((lane % kChunks) ^ swz<D>(r));
    }
  }
  static __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rs, const uint32_t (&off)[kN], int wave, lds_byte* dst) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(dst + (kN * wave + i) * 1024), 16, off[i], 0, 0, 0);
  }
  // Zeros over the rows of this wave's share whose bit in `rows` is clear (the lane overwrites the chunk it
  // loaded itself, so the caller's barrier after the load also covers this).
  static __device__ __forceinline__ void keep(uint64_t rows, int wave, int lane, lds_byte* dst) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (!((rows >> row(wave, lane, i)) & 1)) {
        const half8_t z = {};
        *reinterpret_cast<__attribute__((address_space(3))) half8_t*>(dst + (kN * wave + i) * 1024 + 16 * lane) = z;
      }
  }
};

// A table entry in log2 units.
template <bool BF> __device__ __forceinline__ float table_entry(half_t v) {
  const float e = from_elem<BF>(v), s = e * kLog2e;
  return __builtin_fabsf(e) < INFINITY ? fminf(fmaxf(s, -kTabMax), kTabMax) : s;    // (infinities and NaN as they are)
}
// A head's distance table in LDS: entry x + kTabPad + R holds table[clip(x)] * log2(e), x from -R - kTabPad to R + kTabPad.
template <bool BF>
__device__ __forceinline__ void load_table(const ScoreParams& p, int head, float* tab, int tid, int threads) {
  const int n = 2 * p.radius + 1;
  for (int x = tid; x < n + 2 * kTabPad; x += threads) {
    tab[x] = table_entry<BF>(p.table[(int64_t)head * n + min(max(x - kTabPad, 0), n - 1)]);
  }
}

// Distances lo .. hi of a piece of scores that all clip to one end of the table add one number to each: instead of a
// look-up per score, `add` then goes with the row's constant before the exponential (in log2 units, the scores stay raw).  Ends that
// would swallow a score when added to it (the lowest values of a format, infinities) or are NaN take the look-ups.
struct FarPiece { bool far; float add; };
__device__ __forceinline__ FarPiece far_piece(const ScoreParams& p, const float* tab, int lo, int hi) {
  FarPiece f = {false, 0.f};
  if (hi <= -p.radius || lo >= p.radius) {
    const float end = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, tab[hi <= -p.radius ? 0 : 2 * (p.radius + kTabPad)])));
    if (__builtin_fabsf(end) < 4096.f) { f.far = true; f.add = end; }
  }
  return f;
}

// What one lane knows of its query.
struct LaneRow { int pos, limit, doc; float slope; const float* tab; const half_t* gtab; };

// The rule on 16 scores of the lane's query: s[r] belongs to key jb + 4 g + 8 (r / 4) + r % 4.  Raw
// scores in, what p.cc turns into log2 units out.
__device__ __forceinline__ int key_off(int r) { return 8 * (r >> 2) + (r & 3); }

__device__ __forceinline__ float capped(const ScoreParams& p, float raw) {
  return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(raw * p.k1));
}
__device__ __forceinline__ void cap_scores(const ScoreParams& p, floatx16& s) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = capped(p, s[r]);
}
// The kind of bias is a template argument: behind run-time branches every kind's result is copied to common registers (D
// = 64 without a bias: 32 moves for 190 other vector instructions a tile).  Slopes stay in raw units
// (L.slope has p.slope_mul in it), so that a score costs an addition and a multiply-add.
template <int BIAS>
__device__ __forceinline__ void bias_scores(const ScoreParams& p, const LaneRow& L, int j0 /* jb + 4 g */, floatx16& s) {
  if constexpr (BIAS == kBiasTable) {
    const int x = min(max(j0 - L.pos, -p.radius - kTabPad), p.radius);
    const float* t = L.tab + (x + p.radius + kTabPad);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], p.c, t[key_off(r)]);
  } else if constexpr (BIAS == kBiasSlopes) {
    const float x = (float)(j0 - L.pos);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(__builtin_fabsf(x + (float)key_off(r)), -L.slope, s[r]);
  }
}
__device__ __forceinline__ void limit_scores(const LaneRow& L, int j0, floatx16& s) {
  const int rel = L.limit - j0;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = key_off(r) < rel ? s[r] : -INFINITY;
}
// ids: the documents of the tile's keys in LDS, from key jb + 4 g on
__device__ __forceinline__ void doc_scores(const LaneRow& L, const int* ids, floatx16& s) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = ids[key_off(r)] == L.doc ? s[r] : -INFINITY;
}

// Range number n of a call's B (nq + nk): the blocks of the queries of all samples, then those of the keys; by one wave.
__device__ __forceinline__ void write_doc_range(const ScoreParams& p, int n, int lane) {
  const int nq = (p.Sq + kBlock - 1) / kBlock, nk = (p.Sk + kBlock - 1) / kBlock;
  const bool is_q = n < p.B * nq;
  const int idx = is_q ? n : n - p.B * nq, blocks = is_q ? nq : nk, S = is_q ? p.Sq : p.Sk, b = idx / blocks;
  const DocRange r = doc_range((is_q ? p.docs_q : p.docs_k) + (int64_t)b * S, S, idx - b * blocks, lane);
  if (lane == 0) const_cast<DocRange*>(is_q ? p.dr_q : p.dr_k)[idx] = r;
}

// Document of position i, -1 for none (queries) or -2 (keys), so that they never match.
__device__ __forceinline__ int doc_or(int d, int none) { return d < 0 ? none : d; }
__device__ __forceinline__ int doc_at(const int* docs, int64_t i, bool inside, int none) { return doc_or(inside ? docs[i] : none, none); }

// Host helpers shared by the forward and backward entry points (score_attn_gfx950.hip).
#pragma GCC visibility push(hidden)
int score_attn_check(const void* const* req, int n_req, const int64_t* const* strides, int n_strides, int B, int Hq, int Hkv, int Sq, int Sk, int D,
                     int dtype, float scale, float cap, int radius);
void score_attn_params(ScoreParams& p, const void* q, const void* k, const void* v, const void* table, const void* slopes, const void* prefix,
                       const void* kv_len, const void* docs_q, const void* docs_k, float scale, float cap, int radius, int causal, int q_start,
                       int q_end, const int64_t* qs, const int64_t* ks, const int64_t* vs, int B, int Hq, int Hkv, int Sq, int Sk);
int score_attn_ranges_at(ScoreParams& p, void* ws);      // places the document ranges; how many there are
#pragma GCC visibility pop
