// Linear operator in 8-bit integers for gfx950 (MI355X):
//   stof_quantize_rows_i8   x [M,K] in 16 bits -> int8 with a scale for each row
//   stof_gemm_i8_bias_act   C = act((xq wq^T) sx_m sw_n + bias)
//   stof_linear_i8          both: the user's call on 16-bit activations
//
// A row's scale is a / 127 with a its largest magnitude, a value becomes round(127 x / a), ties to even.
// That rounding is exact for 16-bit inputs: with a' = a 2^-e in [1, 2) and t = 127 x 2^-e (exact: 11 + 7 bits), the
// quotient y = t / a' from one reciprocal and one residual step is within 2^-23 of the true quotient,
// while a quotient of such numbers that is not k + 1/2 lies at least 2^-19 (relative) away from it.
//
// The products are exact: v_mfma_i32_32x32x32_i8 adds into int32, K <= 131056 keeps |sum| below 2^31 for any int8 operands.  The
// only roundings are fp32 scaling, bias and activation, and the store.
//
// Large products use the tile form of the 16-bit GEMM (C^T = W X^T, both operands K-contiguous through LDS
// rows of 128 bytes): a row of 128 bytes now holds 128 of K, so the loads, LDS reads and MFMAs of a tile
// are those of the 16-bit kernel and do twice the arithmetic.  Bound at long K by the LDS reads beside the MFMAs
// (8192^3: 486 us, 2.26 POP/s, MFMA busy 66 %; a library's product 2.08), at K ~ 1024 by what a tile pays beside its
// products: scales and bias are therefore requested ahead of the operands and wait in LDS for the epilogue
// (8192 x 1024 -> 4096 60 -> 53 us, since 44 with single-buffered tiles, 46 with the GELU).  A few tokens use the token form: weights go
// straight to registers, each exactly once, and every workgroup quantises the tokens itself, so a
// single-token projection is one launch.
#include "gemm_tile.h"

namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef unsigned short ushort8_t __attribute__((ext_vector_type(8)));

struct I8Params {
  const half_t* x; const int8_t* xq; const float* sx; const int8_t* wq; const float* sw; const half_t* bias; half_t* out;
  int M, N, K; int64_t ldx, ldq, ldw, ldo;
  int tiles_m, tiles_n;
};

template <int ACT> __device__ __forceinline__ float act_i8(float x) {
  if constexpr (ACT == STOF_ACT_RELU) return x < 0.f ? 0.f : x;    // (keeps the NaN of a row that was not finite)
  else return activate<ACT>(x);
}

// Largest magnitude of 8 values as a bit pattern: the order of the patterns is the order of the magnitudes, with
// infinity and NaN on top.
__device__ __forceinline__ unsigned max_pattern(half8_t v, unsigned m) {
  const ushort8_t u = __builtin_bit_cast(ushort8_t, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (unsigned)(u[e] & 0x7fff));
  return m;
}
// One row's quantiser from its largest pattern.
template <bool BF> struct RowQuant {
  float a, inv, scale; int e; bool finite;
  __device__ __forceinline__ RowQuant(unsigned pattern) {
    finite = pattern < (BF ? 0x7f80u : 0x7c00u);
    const float top = from_elem<BF>(__builtin_bit_cast(half_t, (unsigned short)pattern));
    scale = finite ? top / 127.f : __builtin_nanf("");             // a row that is not finite: zeros times NaN
    e = 0; a = 1.f;
    if (finite && top > 0.f) {
      e = ilogbf(top);
      a = ldexpf(top, -e);
    }
    inv = 1.f / a;
  }
  __device__ __forceinline__ int operator()(half_t v) const {
    const float t = 127.f * __builtin_amdgcn_ldexpf(from_elem<BF>(v), -e);
    float y = t * inv;
    y = __builtin_fmaf(__builtin_fmaf(-y, a, t), inv, y);
    return finite ? (int)__builtin_rintf(y) : 0;
  }
  __device__ __forceinline__ uint64_t pack(half8_t v) const {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half_t a0 = v[i], a1 = v[i + 4];
      lo |= (uint32_t)((*this)(a0) & 255) << (8 * i);
      hi |= (uint32_t)((*this)(a1) & 255) << (8 * i);
    }
    return ((uint64_t)hi << 32) | lo;
  }
};
__device__ __forceinline__ unsigned wave_max_u(unsigned m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
  return m;
}

// One wave per row, 8 values per lane and chunk of 512.  Bound: the reading of x once there are thousands of rows (8192 x 1024
// 7.4 us = 3.4 TB/s, 8192 x 8192 35 us = 5.7 TB/s with the writes), else one trip to memory: rows of up to NV chunks are requested
// at once and stay in registers between the search for the maximum and the rounding (1 x 8192 4.9 us, 8.4 read
// twice; 8192 x 8192 56 us read twice); longer ones (NV = 0) are read again, from the caches.
template <bool BF, int NV>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const half_t* x, int8_t* xq, float* sx, int M, int K, int64_t ldx, int64_t ldq) {
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= M) return;
  const half_t* row = x + m * ldx;
  int8_t* out = xq + m * ldq;
  unsigned top = 0;
  if constexpr (NV > 0) {
    half8_t v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = 512 * i + 8 * lane;
      const half8_t z = {};
      v[i] = k < K ? *reinterpret_cast<const half8_t*>(row + k) : z;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max_pattern(v[i], top);
    const RowQuant<BF> q(wave_max_u(top));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = 512 * i + 8 * lane;
      if (k < K) *reinterpret_cast<uint64_t*>(out + k) = q.pack(v[i]);
    }
    if (lane == 0) sx[m] = q.scale;
  } else {
    for (int k = 8 * lane; k < K; k += 512) top = max_pattern(*reinterpret_cast<const half8_t*>(row + k), top);
    const RowQuant<BF> q(wave_max_u(top));
    for (int k = 8 * lane; k < K; k += 512) *reinterpret_cast<uint64_t*>(out + k) = q.pack(*reinterpret_cast<const half8_t*>(row + k));
    if (lane == 0) sx[m] = q.scale;
  }
}

__device__ __forceinline__ intx16 mfma_i8(int4_t a, int4_t b, intx16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int4_t lds_frag_i8(const lds_byte* tile, int off) {
  return *reinterpret_cast<const __attribute__((address_space(3))) int4_t*>(tile + off);
}

// ---- tile form: T x T output tile, WM x WN waves, each T/WM tokens x T/WN features; K tiles of 128 through ST buffers.
// KG > 1: KG groups of WM x WN waves take every KG-th K tile each, through buffers of their own, and their integer
// sums are added at the end (exact, so their order does not matter).
constexpr int kI8K = 128;

template <int ACT, bool BF, int T, int WM, int WN, int ST, int KG, int OCC>
__global__ __launch_bounds__(64 * WM * WN * KG, OCC) void gemm_i8_kernel(const I8Params p) {
  constexpr int kTile = T * kI8K;
  constexpr int kLoads = T / 8 / (WM * WN); // load instructions per wave and operand tile (8 rows each)
  constexpr int kTok = T / WM / 32, kFeat = T / WN / 32;   // 32-wide MFMA tiles per wave and direction
  __shared__ __attribute__((aligned(1024))) unsigned char a0_all[KG * kTile];
  __shared__ __attribute__((aligned(1024))) unsigned char w0_all[KG * kTile];
  __shared__ __attribute__((aligned(1024))) unsigned char a1_all[ST == 2 ? KG * kTile : 16];
  __shared__ __attribute__((aligned(1024))) unsigned char w1_all[ST == 2 ? KG * kTile : 16];

  const int group = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / (64 * WM * WN)));
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) % (WM * WN));
  lds_byte* a0 = (lds_byte*)a0_all + group * kTile; lds_byte* w0 = (lds_byte*)w0_all + group * kTile;
  lds_byte* a1 = (lds_byte*)a1_all + (ST == 2 ? group * kTile : 0); lds_byte* w1 = (lds_byte*)w1_all + (ST == 2 ? group * kTile : 0);
  const int lane = threadIdx.x & 63, j32 = lane & 31, g = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  __shared__ __attribute__((aligned(16))) float sx_lds[T], sw_lds[T], b_lds[T];
  int tm, tn;
  if (p.tiles_m < 8) {                      // (the raster gives token tile tm to XCD tm % 8: fewer would leave XCDs empty)
    tn = blockIdx.x / p.tiles_m;
    tm = blockIdx.x - tn * p.tiles_m;
  } else if (!raster_tile((int)blockIdx.x, p.tiles_m, p.tiles_n, tm, tn)) {
    return;
  }
  const int m0 = tm * T, n0 = tn * T;
  // the epilogue's scales and bias: requested ahead of the operands, into LDS once the products are done
  const int et = threadIdx.x % T;
  const float e_sx = p.sx[min(m0 + et, p.M - 1)], e_sw = p.sw[min(n0 + et, p.N - 1)];
  const float e_b = p.bias ? from_elem<BF>(p.bias[min(n0 + et, p.N - 1)]) : 0.f;

  // rows past the edge re-read the last row; in the last K tile, chunks past K lie beyond the resource's
  // extent and arrive as zeros
  constexpr uint32_t kOut = 0x80000000u;
  uint32_t a_off[kLoads], w_off[kLoads];
  int chunk_k[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = 8 * (kLoads * wave + i) + (lane >> 3);
    const int chunk = (lane & 7) ^ swz(r);
    chunk_k[i] = 16 * chunk;
    a_off[i] = (uint32_t)min(r, p.M - 1 - m0) * (uint32_t)p.ldq + 16 * chunk;
    w_off[i] = (uint32_t)min(r, p.N - 1 - n0) * (uint32_t)p.ldw + 16 * chunk;
  }
  const __amdgpu_buffer_rsrc_t a_rs = stof_wave_rsrc(p.xq + (int64_t)m0 * p.ldq), w_rs = stof_wave_rsrc(p.wq + (int64_t)n0 * p.ldw);
  auto issue = [&](int kt, lds_byte* ad, lds_byte* wd) {
    const uint32_t koff = (uint32_t)kt * kI8K;
    const int left = p.K - kt * kI8K;
    if (left >= kI8K) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) dma16b(a_rs, a_off[i], koff, ad + (kLoads * wave + i) * 1024);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) dma16b(w_rs, w_off[i], koff, wd + (kLoads * wave + i) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) dma16b(a_rs, chunk_k[i] < left ? a_off[i] : kOut, koff, ad + (kLoads * wave + i) * 1024);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) dma16b(w_rs, chunk_k[i] < left ? w_off[i] : kOut, koff, wd + (kLoads * wave + i) * 1024);
    }
  };
  int rd[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) rd[ks] = j32 * kI8K + (((2 * ks + g) ^ swz(j32)) << 4);

  intx16 acc[kFeat][kTok];                  // [feature tile][token tile]
#pragma unroll
  for (int i = 0; i < kFeat; ++i)
#pragma unroll
    for (int j = 0; j < kTok; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  auto compute = [&](const lds_byte* at, const lds_byte* wt) {
    int4_t xa[2][kTok], wb[2][kFeat];
    auto fetch = [&](int ks, int set) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) xa[set][i] = lds_frag_i8(at, (T / WM * wm + 32 * i) * kI8K + rd[ks]);
#pragma unroll
      for (int i = 0; i < kFeat; ++i) wb[set][i] = lds_frag_i8(wt, (T / WN * wn + 32 * i) * kI8K + rd[ks]);
    };
    fetch(0, 0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks + 1 < 4) fetch(ks + 1, (ks + 1) & 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ni = 0; ni < kFeat; ++ni)
#pragma unroll
        for (int mi = 0; mi < kTok; ++mi) acc[ni][mi] = mfma_i8(wb[ks & 1][ni], xa[ks & 1][mi], acc[ni][mi]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // group's K tiles: group, group + KG, ...; every group passes every barrier
  const int nk = (p.K + kI8K - 1) / kI8K, steps = (nk + KG - 1) / KG;
  auto tile = [&](int i) { return i * KG + group; };
  if (tile(0) < nk) issue(tile(0), a0, w0);
  if constexpr (ST == 1) {
    for (int i = 0; i < steps; ++i) {
      __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt(0): this wave's share of the tile landed
      __syncthreads();
      if (tile(i) < nk) compute(a0, w0);
      __syncthreads();
      if (i + 1 < steps && tile(i + 1) < nk) issue(tile(i + 1), a0, w0);
    }
  } else {
    for (int i = 0; i < steps; i += 2) {
      __builtin_amdgcn_s_waitcnt(0x0F70);
      __syncthreads();
      if (tile(i + 1) < nk) issue(tile(i + 1), a1, w1);
      if (tile(i) < nk) compute(a0, w0);
      if (i + 1 < steps) {
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
        if (tile(i + 2) < nk) issue(tile(i + 2), a0, w0);
        if (tile(i + 1) < nk) compute(a1, w1);
      }
    }
  }
  if ((int)threadIdx.x < T) { sx_lds[et] = e_sx; sw_lds[et] = e_sw; b_lds[et] = e_b; }
  __syncthreads();                          // every wave is done with the operand tiles
  if constexpr (KG > 1) {
    // the other groups' sums to group 0, T T / (64 WM WN) integers per lane through the operand tiles
    constexpr int kInts = kFeat * kTok * 16;
    static_assert(64 * WM * WN * kInts * 4 <= 2 * kTile, "a group's sums fit its two operand buffers");
#pragma unroll
    for (int n = 0; n < kInts; ++n) {
      lds_byte* at = ((n < kInts / 2) ? a0 : w0) + ((n % (kInts / 2)) * (WM * WN) + wave) * 256 + 4 * lane;
      if (group > 0) *reinterpret_cast<__attribute__((address_space(3))) int*>(at) = acc[n / (16 * kTok)][(n / 16) % kTok][n % 16];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int n = 0; n < kInts; ++n)
#pragma unroll
      for (int o = 1; o < KG; ++o)
        acc[n / (16 * kTok)][(n / 16) % kTok][n % 16] += *reinterpret_cast<const __attribute__((address_space(3))) int*>(
            ((n < kInts / 2) ? a0 : w0) + o * kTile + ((n % (kInts / 2)) * (WM * WN) + wave) * 256 + 4 * lane);
  }

  // epilogue: 32 tokens x (T / WN) features at a time through the wave's own LDS rows (kFeat * 64 bytes, 16-byte chunks
  // XOR-ed by the row) and out in whole rows
  constexpr int kRow = kFeat * 64, kC = kRow / 16;
  lds_byte* stage = a0 + wave * (32 * kRow);   // (group 0's own)
  const int m_base = m0 + T / WM * wm, n_base = n0 + T / WN * wn;
  const __amdgpu_buffer_rsrc_t o_rs = stof_wave_rsrc(p.out + (int64_t)m_base * p.ldo + n_base);
#pragma unroll
  for (int mi = 0; mi < kTok; ++mi) {
    const float sx = sx_lds[T / WM * wm + 32 * mi + j32];
#pragma unroll
    for (int ni = 0; ni < kFeat; ++ni)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int n = T / WN * wn + 32 * ni + 8 * q4 + 4 * g;
        const floatx4 sw = *reinterpret_cast<const floatx4*>(sw_lds + n), bv = *reinterpret_cast<const floatx4*>(b_lds + n);
        half4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = to_elem<BF>(act_i8<ACT>(__builtin_fmaf((float)acc[ni][mi][4 * q4 + e], sx * sw[e], bv[e])));
        *reinterpret_cast<__attribute__((address_space(3))) half4_t*>(stage + j32 * kRow + (((4 * ni + q4) ^ (j32 & (kC - 1))) << 4) + 8 * g) = o;
      }
#pragma unroll
    for (int i = 0; i < 32 * kC / 64; ++i) {
      const int t = (64 / kC) * i + lane / kC, c = lane % kC;
      const half8_t o = lds_frag(stage, t * kRow + ((c ^ (t & (kC - 1))) << 4));
      if (m_base + 32 * mi + t < p.M && n_base + 8 * c < p.N)
        stof_store16_through(o_rs, (uint32_t)(32 * mi + t) * (uint32_t)(p.ldo * 2) + 16 * c, o);
    }
  }
}

// ---- token form: up to 16 tokens, 16 features at a time per workgroup, K split over the four waves.
// v_mfma_i32_16x16x64_i8: A = 16 weight rows (lane & 15) x 64 of K (16 bytes per lane, group lane >> 4), B = the tokens from
// LDS.  Result: token lane & 15, features 4 (lane >> 4) + r.  A wave's weights arrive in rounds of kTokLoads loads, the
// next round (of the next 16 features, too) requested before the products of the current one.
//
// Bound: the weights for one token, quantising for many, which every workgroup does for itself: from two tokens on
// each wave takes whole rows (registers hold them between the search for the maximum and the rounding; the waves
// sharing every row: 16 x 1024 -> 4096 16.9 us, so 8.6), and a workgroup takes every gridDim-th block of 16 features (16 x 1024
// -> 16384 23.2 -> 12.5).  Against a quantising launch and the tile form, whose gap of 2 us is not in these figures: 1 x
// 1024 -> 4096 4.2 | 8.3 us, 1 x 4096 -> 4096 8.8 | 13.0, 16 x 1024 -> 4096 8.6 | 8.9, 8 x 4096 -> 4096 12.3 | 13.8, 1 x 4096 -> 16384
// 20.3 | 17.9; 16 x 4096 -> 4096 17.5 | 14.2, so rows beyond 64 KB of LDS take two launches.
constexpr int kTokMax = 16;
constexpr int kTokLoads = 8;
constexpr int kTokLds = 64 * 1024;
constexpr int kTokGrid = 512;
constexpr int kTokKeep = 8;        // chunks of 512 values of a row in registers

template <int ACT, bool BF>
__global__ __launch_bounds__(256) void linear_i8_token_kernel(const I8Params p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char xq_lds[];       // [M][Kp + 16], Kp = K rounded up to 64, zeros beyond K
  __shared__ unsigned tops[4];
  __shared__ float sxs[kTokMax];
  __shared__ int sums[2][4][16][17];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
  const int steps = (p.K + 63) / 64, Kp = steps * 64, pitch = Kp + 16, blocks = (p.N + 15) / 16;
  const int mine = (steps - wave + 3) / 4;
  auto k_of = [&](int s) { return 64 * (4 * s + wave) + 16 * kg; };          // this wave's step s
  auto weights = [&](int block, int s) -> int4_t {
    const int k = k_of(s);
    return *reinterpret_cast<const int4_t*>(p.wq + (int64_t)min(16 * block + row, p.N - 1) * p.ldw + (k < p.K ? k : 0));   // (times zeros of x beyond K)
  };
  int block = blockIdx.x;
  int4_t wa[kTokLoads];
#pragma unroll
  for (int i = 0; i < kTokLoads; ++i) wa[i] = i < mine ? weights(block, i) : int4_t{0, 0, 0, 0};

  if (p.M == 1) {          // the waves share the row
    unsigned top = 0;
    for (int k = 8 * threadIdx.x; k < p.K; k += 2048) top = max_pattern(*reinterpret_cast<const half8_t*>(p.x + k), top);
    top = wave_max_u(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    const RowQuant<BF> q(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    for (int k = 8 * threadIdx.x; k < Kp; k += 2048)
      *reinterpret_cast<uint64_t*>(xq_lds + k) = k < p.K ? q.pack(*reinterpret_cast<const half8_t*>(p.x + k)) : 0;
    if (threadIdx.x == 0) sxs[0] = q.scale;
  } else {
    for (int m = wave; m < p.M; m += 4) {
      const half_t* src = p.x + m * p.ldx;
      half8_t v[kTokKeep];
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < kTokKeep; ++i) {
        const int k = 512 * i + 8 * lane;
        const half8_t z = {};
        v[i] = k < p.K ? *reinterpret_cast<const half8_t*>(src + k) : z;
      }
#pragma unroll
      for (int i = 0; i < kTokKeep; ++i) top = max_pattern(v[i], top);
      for (int k = 512 * kTokKeep + 8 * lane; k < p.K; k += 512) top = max_pattern(*reinterpret_cast<const half8_t*>(src + k), top);
      const RowQuant<BF> q(wave_max_u(top));
#pragma unroll
      for (int i = 0; i < kTokKeep; ++i) {
        const int k = 512 * i + 8 * lane;
        if (k < Kp) *reinterpret_cast<uint64_t*>(xq_lds + m * pitch + k) = q.pack(v[i]);      // (zeros beyond K)
      }
      for (int k = 512 * kTokKeep + 8 * lane; k < Kp; k += 512)
        *reinterpret_cast<uint64_t*>(xq_lds + m * pitch + k) = k < p.K ? q.pack(*reinterpret_cast<const half8_t*>(src + k)) : 0;
      if (lane == 0) sxs[m] = q.scale;
    }
  }
  __syncthreads();

  const unsigned char* xrow = xq_lds + min(row, p.M - 1) * pitch;
  // thread (token t, feature f) of the epilogue
  const int t = threadIdx.x >> 4, f = threadIdx.x & 15;
  for (int it = 0; block < blocks; ++it) {
    const int next = block + gridDim.x;
    int4_t acc = {0, 0, 0, 0};
    for (int s0 = 0; s0 < mine; s0 += kTokLoads) {
      const bool last = s0 + kTokLoads >= mine;
      int4_t wn[kTokLoads];
#pragma unroll
      for (int i = 0; i < kTokLoads; ++i) {
        const int s = last ? i : s0 + kTokLoads + i;
        wn[i] = s < mine && (!last || next < blocks) ? weights(last ? next : block, s) : int4_t{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < kTokLoads; ++i)
        if (s0 + i < mine) {
          const int4_t xb = *reinterpret_cast<const int4_t*>(xrow + k_of(s0 + i));
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa[i], xb, acc, 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < kTokLoads; ++i) wa[i] = wn[i];
    }
    // (two sets of sums in turn: a set is written again only behind the barrier of the block between)
    int (*part)[16][17] = sums[it & 1];
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][row][4 * kg + r] = acc[r];
    __syncthreads();
    const int n = 16 * block + f;
    if (t < p.M && n < p.N) {
      const int total = (part[0][t][f] + part[1][t][f]) + (part[2][t][f] + part[3][t][f]);
      const float b = p.bias ? from_elem<BF>(p.bias[n]) : 0.f;
      p.out[(int64_t)t * p.ldo + n] = to_elem<BF>(act_i8<ACT>(__builtin_fmaf((float)total, sxs[t] * p.sw[n], b)));
    }
    block = next;
  }
}

int64_t token_pitch(int64_t K) { return (K + 63) / 64 * 64 + 16; }
bool token_form(int64_t M, int64_t K) { return M <= kTokMax && M * token_pitch(K) <= kTokLds; }
int64_t padded(int64_t K) { return (K + 15) / 16 * 16; }

// Which tile form, by the number of tiles and the length of K (us, form taken | its neighbour):
//  * 128 x 128 tiles that leave half the device empty -> 64 x 64, and with few of those and a long K four groups of
//    waves along K: 777 x 768 -> 2304 7.6 | 9.1 (128), 512 x 4096 -> 1024 12.3 | 18.3 (64 without groups),
//    100 x 4096 -> 4096 11.6 | 17.5, 2048 x 4096 -> 1024 (512 tiles of 64) 19.9 | 23.3 (groups), K 1024 even;
//  * 256 x 256 (0.75 KB of LDS reads per MFMA instead of 1 KB, one workgroup per unit) needs every unit busy and a K
//    that outweighs its unoverlapped epilogue: 8192^3 489 | 530, 4096^3 66.6 | 72.4, 8192 x 1024 -> 4096 50 | 46;
//  * 128 x 128 with two buffers while all tiles are resident (two per unit): 8192 x 4096 -> 1024 38 | 46; with one
//    buffer, four workgroups per unit whose epilogues and products overlap, beyond: 8192 x 1024 -> 4096 46 | 53,
//    65536 x 1024 -> 1024 94 | 103.
enum { kTile64, kTile64Groups, kTile128, kTile128Single, kTile256 };
int tile_form(int64_t M, int64_t N, int64_t K) {
  const int64_t t64 = ((M + 63) / 64) * ((N + 63) / 64), t128 = ((M + 127) / 128) * ((N + 127) / 128), t256 = ((M + 255) / 256) * ((N + 255) / 256);
  if (t128 < 256) return t64 <= 256 && K >= 2048 ? kTile64Groups : kTile64;
  if (K >= 2048 && t256 >= 256) return kTile256;
  return t128 <= 512 ? kTile128 : kTile128Single;
}

template <int ACT, bool BF>
void launch_gemm(I8Params& p, hipStream_t st) {
  const int form = tile_form(p.M, p.N, p.K);
  const int T = form == kTile256 ? 256 : form >= kTile128 ? 128 : 64;
  p.tiles_m = (p.M + T - 1) / T;
  p.tiles_n = (p.N + T - 1) / T;
  const dim3 grid(p.tiles_m < 8 ? (unsigned)(p.tiles_m * p.tiles_n) : raster_grid(p.tiles_m, p.tiles_n));
  switch (form) {
    case kTile64: gemm_i8_kernel<ACT, BF, 64, 2, 2, 2, 1, 4><<<grid, dim3(256), 0, st>>>(p); break;
    case kTile64Groups: gemm_i8_kernel<ACT, BF, 64, 2, 2, 2, 4, 1><<<grid, dim3(1024), 0, st>>>(p); break;
    case kTile128: gemm_i8_kernel<ACT, BF, 128, 2, 2, 2, 1, 2><<<grid, dim3(256), 0, st>>>(p); break;
    case kTile128Single: gemm_i8_kernel<ACT, BF, 128, 2, 2, 1, 1, 4><<<grid, dim3(256), 0, st>>>(p); break;
    default: gemm_i8_kernel<ACT, BF, 256, 2, 4, 2, 1, 1><<<grid, dim3(512), 0, st>>>(p); break;
  }
}
template <int ACT, bool BF>
void launch_token(I8Params& p, hipStream_t st) {
  const size_t lds = (size_t)p.M * (size_t)token_pitch(p.K);
  linear_i8_token_kernel<ACT, BF><<<dim3((unsigned)min((p.N + 15) / 16, kTokGrid)), dim3(256), lds, st>>>(p);
}
template <bool BF>
void launch_act(I8Params& p, int act, bool token, hipStream_t st) {
  switch (act) {
    case STOF_ACT_NONE: token ? launch_token<STOF_ACT_NONE, BF>(p, st) : launch_gemm<STOF_ACT_NONE, BF>(p, st); break;
    case STOF_ACT_GELU_ERF: token ? launch_token<STOF_ACT_GELU_ERF, BF>(p, st) : launch_gemm<STOF_ACT_GELU_ERF, BF>(p, st); break;
    case STOF_ACT_GELU_TANH: token ? launch_token<STOF_ACT_GELU_TANH, BF>(p, st) : launch_gemm<STOF_ACT_GELU_TANH, BF>(p, st); break;
    default: token ? launch_token<STOF_ACT_RELU, BF>(p, st) : launch_gemm<STOF_ACT_RELU, BF>(p, st); break;
  }
}
template <bool BF>
void launch_quantize_nv(const half_t* x, int8_t* xq, float* sx, int M, int K, int64_t ldx, int64_t ldq, hipStream_t st) {
  const dim3 grid((unsigned)((M + 3) / 4)), block(256);
  if (K <= 1024) quantize_rows_kernel<BF, 2><<<grid, block, 0, st>>>(x, xq, sx, M, K, ldx, ldq);
  else if (K <= 4096) quantize_rows_kernel<BF, 8><<<grid, block, 0, st>>>(x, xq, sx, M, K, ldx, ldq);
  else if (K <= 8192) quantize_rows_kernel<BF, 16><<<grid, block, 0, st>>>(x, xq, sx, M, K, ldx, ldq);
  else if (K <= 16384) quantize_rows_kernel<BF, 32><<<grid, block, 0, st>>>(x, xq, sx, M, K, ldx, ldq);
  else quantize_rows_kernel<BF, 0><<<grid, block, 0, st>>>(x, xq, sx, M, K, ldx, ldq);
}
void launch_quantize(const void* x, int8_t* xq, float* sx, int M, int K, int64_t ldx, int64_t ldq, int dtype, hipStream_t st) {
  if (dtype == STOF_DTYPE_BF16) launch_quantize_nv<true>((const half_t*)x, xq, sx, M, K, ldx, ldq, st);
  else launch_quantize_nv<false>((const half_t*)x, xq, sx, M, K, ldx, ldq, st);
}

int check_sizes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 16 != 0 || N % 8 != 0) return STOF_ERR_BAD_SHAPE;
  if (M > (1 << 28) || N > (1 << 28) || K > 131056 || ((M + 63) / 64 + 8) * ((N + 63) / 64) > 0x0fffffff) return STOF_ERR_BAD_SHAPE;
  if (dtype != STOF_DTYPE_F16 && dtype != STOF_DTYPE_BF16) return STOF_ERR_UNSUPPORTED;
  return STOF_OK;
}
int check_common(const void* wq, const float* sw, const void* bias, const void* out, int64_t K, int64_t N, int64_t ldw, int64_t ldo, int act) {
  if (!wq || !sw || !out) return STOF_ERR_NULL_POINTER;
  if (!stof_aligned16(wq) || !stof_aligned16(sw) || !stof_aligned16(out) || (bias && !stof_aligned16(bias))) return STOF_ERR_MISALIGNED;
  if (ldw < K || ldo < N || ldw > (1 << 23) || ldo > (1 << 22)) return STOF_ERR_BAD_SHAPE;    // 256 rows of a tile stay below 2^31 bytes
  if (ldw % 16 != 0 || ldo % 8 != 0) return STOF_ERR_MISALIGNED;
  if (act < STOF_ACT_NONE || act > STOF_ACT_RELU) return STOF_ERR_UNSUPPORTED;
  return STOF_OK;
}

}  // namespace

extern "C" int stof_quantize_rows_i8(const void* x, int8_t* xq, float* sx, int64_t M, int64_t K, int64_t ldx, int64_t ldq, int dtype, void* stream) {
  const int rc = check_sizes(M, 8, K, dtype);
  if (rc) return rc;
  if (!x || !xq || !sx) return STOF_ERR_NULL_POINTER;
  if (!stof_aligned16(x) || !stof_aligned16(xq) || ldx % 8 != 0 || ldq % 16 != 0) return STOF_ERR_MISALIGNED;
  if (ldx < K || ldq < K) return STOF_ERR_BAD_SHAPE;
  launch_quantize(x, xq, sx, (int)M, (int)K, ldx, ldq, dtype, (hipStream_t)stream);
  return stof_check_launch();
}

extern "C" int stof_gemm_i8_bias_act(const int8_t* xq, const float* sx, const int8_t* wq, const float* sw, const void* bias, void* out,
                                     int64_t M, int64_t N, int64_t K, int64_t ldq, int64_t ldw, int64_t ldo, int act, int dtype, void* stream) {
  int rc = check_sizes(M, N, K, dtype);
  if (rc) return rc;
  rc = check_common(wq, sw, bias, out, K, N, ldw, ldo, act);
  if (rc) return rc;
  if (!xq || !sx) return STOF_ERR_NULL_POINTER;
  if (!stof_aligned16(xq) || ldq % 16 != 0) return STOF_ERR_MISALIGNED;
  if (ldq < K || ldq > (1 << 23)) return STOF_ERR_BAD_SHAPE;
  I8Params p = {};
  p.xq = xq; p.sx = sx; p.wq = wq; p.sw = sw; p.bias = (const half_t*)bias; p.out = (half_t*)out;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.ldq = ldq; p.ldw = ldw; p.ldo = ldo;
  if (dtype == STOF_DTYPE_BF16) launch_act<true>(p, act, false, (hipStream_t)stream);
  else launch_act<false>(p, act, false, (hipStream_t)stream);
  return stof_check_launch();
}

extern "C" int64_t stof_linear_i8_workspace_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || token_form(M, K)) return 0;
  return M * padded(K) + (M * 4 + 15) / 16 * 16;
}

extern "C" int stof_linear_i8(const void* x, const int8_t* wq, const float* sw, const void* bias, void* out,
                              int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldo, int act, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K, dtype);
  if (rc) return rc;
  rc = check_common(wq, sw, bias, out, K, N, ldw, ldo, act);
  if (rc) return rc;
  if (!x) return STOF_ERR_NULL_POINTER;
  if (!stof_aligned16(x) || ldx % 8 != 0) return STOF_ERR_MISALIGNED;
  if (ldx < K) return STOF_ERR_BAD_SHAPE;
  const bool token = token_form(M, K);
  I8Params p = {};
  if (!token) {
    if (!workspace) return STOF_ERR_NULL_POINTER;
    if (!stof_aligned16(workspace)) return STOF_ERR_MISALIGNED;
    if (workspace_bytes < stof_linear_i8_workspace_bytes(M, K)) return STOF_ERR_BAD_SHAPE;
    p.ldq = padded(K);
    p.xq = (int8_t*)workspace;
    p.sx = (float*)((char*)workspace + M * p.ldq);
    launch_quantize(x, (int8_t*)p.xq, (float*)p.sx, (int)M, (int)K, ldx, p.ldq, dtype, (hipStream_t)stream);
  }
  p.x = (const half_t*)x; p.wq = wq; p.sw = sw; p.bias = (const half_t*)bias; p.out = (half_t*)out;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.ldx = ldx; p.ldw = ldw; p.ldo = ldo;
  if (dtype == STOF_DTYPE_BF16) launch_act<true>(p, act, token, (hipStream_t)stream);
  else launch_act<false>(p, act, token, (hipStream_t)stream);
  return stof_check_launch();
}
