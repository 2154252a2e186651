// layer_norm.hip -- layer norm over the channels of a row and its backward pass.
//
//   forward    mean = sum(x) / D, var = sum((x - mean)^2) / D, rstd = 1 / sqrt(var + eps), y = (x - mean) rstd w + b
//   backward   g = dy w, xh = (x - mean) rstd:   dx = rstd (g - sum(g) / D - xh sum(g xh) / D),   dw = sum over rows of dy xh,
//              db = sum over rows of dy
//
// Bound by HBM: x in, y out (forward); x and dy in, dx out (backward).  A row is read ONCE and stays in registers between its sums and
// its output: LPR lanes hold NV pieces of 16 bytes each.  The backward pass keeps the two weight gradients of its lanes' columns in f32
// registers over all the rows that a workgroup takes, so they cost one partial row pair per workgroup and a second, small launch that
// adds those in a fixed order: no atomics, the same bits on every run.  All sums are f32; every output is rounded once.
// Measured (copies of this size run at 5.0 .. 5.4 TB/s): forward 16384 x 4096 bf16 46 us = 5.8 TB/s (parts of it stay in the caches), 230400 x
// 128 f16 20 us = 6.0; backward 81 us = 5.0 TB/s and 36 us = 4.9.  f32: forward 8192 x 4096 44 us = 6.1 TB/s, 30000 x 771 35 us = 5.3, 2048 x 16384
// 49 us = 5.5; backward 77 us = 5.3 TB/s, 53 us = 5.3, 93 us = 4.3 (sixteen waves of four pieces a lane: no row fetched ahead).
#include "rows.h"

#define LN_MAX_COLS 16384

// sum over the LPR lanes of a row, LPR <= 64: every lane gets it.  DPP adds within 16 lanes (common.h), two exchanges beyond.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  if (LPR >= 2) v = dpp_add<0xB1, 0xf>(v);
  if (LPR >= 4) v = dpp_add<0x4E, 0xf>(v);
  if (LPR >= 8) v = dpp_add<0x141, 0xf>(v);
  if (LPR >= 16) v = dpp_add<0x140, 0xf>(v);
  if (LPR >= 32) v += __shfl_xor(v, 16, 64);
  if (LPR >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// two sums over the lanes of a row.  LPR > 64: the workgroup's waves meet in LDS; callers use two buffers in turn, so that one barrier
// per call is enough (a wave writes a buffer again only behind the barrier of the call in between).
template <int LPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*red)[2]) {
  a = lanes_sum<(LPR < 64 ? LPR : 64)>(a);
  b = lanes_sum<(LPR < 64 ? LPR : 64)>(b);
  if (LPR > 64) {
    constexpr int W = LPR / 64;
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][0] = a;
      red[threadIdx.x >> 6][1] = b;
    }
    lds_barrier();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < W; i++) {
      a += red[i][0];
      b += red[i][1];
    }
  }
}

// columns [c, c + V) of a piece and how many of them the piece before it owns: the last piece of a row ends with the row and overlaps its
// neighbour where D is no multiple of V.  Both lanes form and store the same bits there; a row's sums leave the first `skip` out.  skip >= V:
// no piece (its lane reads the last one).  Pieces cut off element by element cost more (32768 x 1500 bf16: forward 53 instead of 38 us,
// backward 106 instead of 63).  whole: known not to be the last.
template <int V>
__device__ __forceinline__ void ln_piece(int piece, int D, int& c, int& skip, bool whole = false) {
  c = whole ? piece * V : min(piece * V, D - V);
  skip = whole ? 0 : piece * V - c;
}

template <int LPR>
constexpr int ln_block() { return LPR > 64 ? LPR : 256; }

// ---------------------------------------------------------------------------------------------
// forward.  Two sums over the row, in turn: the mean, then sum d and sum d^2 of the deviations d = x - mean.  The first of these is what
// rounding left of the mean; taking it out again keeps the deviations exact where |mean| is far above the row's spread.  The stored mean is the
// corrected one: closer than the first where |mean| is above the spread (f32 rows of 128: 5e-8 of the mean at most against 1.2e-7).  Where it is
// below and the first sum was exact (f16 rows of 128), the correction is nothing but the deviations' rounding, and the stored mean is off by 2^-24 of
// the spread where the first alone would be right -- what the output's own deviations carry anyway.
// ---------------------------------------------------------------------------------------------
template <typename T, typename W, int V, int LPR, int NV>
__global__ __launch_bounds__(ln_block<LPR>()) void layer_norm_fwd_kernel(const T* __restrict__ x, long xstride, const W* __restrict__ w,
                                                                         const W* __restrict__ b, T* __restrict__ y,
                                                                         float* __restrict__ mean, float* __restrict__ rstd, long n, int D,
                                                                         float inv_d, float eps) {
  constexpr int ROWS = ln_block<LPR>() / LPR;
  __shared__ float red[2][LPR > 64 ? LPR / 64 : 1][2];   // (per sum: the other sum's barrier lies between two uses)
  const int lane = threadIdx.x % LPR;
  const long step = (long)gridDim.x * ROWS;
  RowPiece<W, V> wp[NV], bp[NV];
  int c[NV], skip[NV];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    ln_piece<V>(j * LPR + lane, D, c[j], skip[j], j < NV / 2);
    if (w) wp[j] = row_get<W, V>(w + c[j]);
    if (b) bp[j] = row_get<W, V>(b + c[j]);
  }
  for (long r = (long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / LPR : 0); r < n; r += step) {
    RowPiece<T, V> p[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) p[j] = row_get<T, V>(x + r * xstride + c[j]);
    float f[NV][V], s = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        f[j][i] = (float)p[j].e[i];
        s += i >= skip[j] ? f[j][i] : 0.0f;
      }
    row_sum2<LPR>(s, q, red[0]);
    const float m1 = s * inv_d;
    s = q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        f[j][i] -= m1;
        const float d = i >= skip[j] ? f[j][i] : 0.0f;
        s += d;
        q += d * d;
      }
    row_sum2<LPR>(s, q, red[1]);
    const float m2 = s * inv_d, v0 = q * inv_d - m2 * m2, var = v0 < 0.0f ? 0.0f : v0, rs = 1.0f / sqrtf(var + eps);   // (a NaN stays)
    if (lane == 0 && mean) {
      mean[r] = m2 == m2 ? m1 + m2 : m1;                        // (an infinity in the row: the mean is one, m2 is a NaN)
      rstd[r] = rs;
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        float v = (f[j][i] - m2) * rs;
        if (w) v *= (float)wp[j].e[i];
        if (b) v += (float)bp[j].e[i];
        f[j][i] = v;
      }
      if (skip[j] < V) row_put<T, V, false>(y + r * D + c[j], f[j]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// backward.  part: [workgroups][2][D] f32 (dw | db), or nullptr: neither is asked for.  dweight / dbias: nullptr where that one is not.
//
// FEW: few rows, one launch, no part.  The weight gradients are formed by further workgroups (from row_blocks on), ln_columns pieces of the
// columns each over all rows, which are read a second time (they lie in the caches): dw and db need no sum over a row, mean and rstd are given.
// ---------------------------------------------------------------------------------------------
template <int BLOCK>
constexpr int ln_columns() { return BLOCK > 256 ? BLOCK / 64 : 4; }    // 32 or 64 lanes share a piece's rows

template <typename T, typename W, int V, int BLOCK>
__device__ __forceinline__ void layer_norm_columns(const T* __restrict__ dy, long dstride, const T* __restrict__ x, long xstride,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd, W* __restrict__ dweight,
                                                   W* __restrict__ dbias, int n, int D, int block, float* __restrict__ red) {
  constexpr int COLUMNS = ln_columns<BLOCK>(), SUBS = BLOCK / COLUMNS, WAVES = BLOCK / 64;
  const int piece = threadIdx.x % COLUMNS, wave = threadIdx.x / 64;
  int c, skip;
  ln_piece<V>(block * COLUMNS + piece, D, c, skip);
  float sum[2][V];                                               // dw | db
#pragma unroll
  for (int i = 0; i < V; i++) sum[0][i] = sum[1][i] = 0.0f;
  if (skip < V) {
#pragma unroll 4
    for (int r = threadIdx.x / COLUMNS; r < n; r += SUBS) {
      const RowPiece<T, V> p = row_get<T, V>(x + (long)r * xstride + c), d = row_get<T, V>(dy + (long)r * dstride + c);
      const float mu = mean[r], rs = rstd[r];
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float u = (float)d.e[i];
        sum[0][i] += u * (((float)p.e[i] - mu) * rs);
        sum[1][i] += u;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int i = 0; i < V; i++) {
#pragma unroll
      for (int o = 32; o >= COLUMNS; o >>= 1) sum[k][i] += __shfl_down(sum[k][i], o, 64);
      if (threadIdx.x % 64 < COLUMNS) red[((wave * 2 + k) * COLUMNS + piece) * V + i] = sum[k][i];
    }
  __syncthreads();
  if (threadIdx.x < 2 * COLUMNS) {
    const int k = threadIdx.x / COLUMNS;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      acc[i] = 0.0f;
#pragma unroll
      for (int q = 0; q < WAVES; q++) acc[i] += red[((q * 2 + k) * COLUMNS + piece) * V + i];
    }
    W* out = k ? dbias : dweight;
    if (skip < V && out) row_put<W, V, false>(out + c, acc);
  }
}

template <typename T, typename W, int V, int LPR, int NV, bool FEW>
__global__ __launch_bounds__(ln_block<LPR>()) void layer_norm_bwd_kernel(const T* __restrict__ dy, long dstride, const T* __restrict__ x,
                                                                         long xstride, const float* __restrict__ mean,
                                                                         const float* __restrict__ rstd, const W* __restrict__ w,
                                                                         T* __restrict__ dx, float* __restrict__ part, W* __restrict__ dweight,
                                                                         W* __restrict__ dbias, long n, int D, float inv_d, int row_blocks) {
  constexpr int BLOCK = ln_block<LPR>(), ROWS = BLOCK / LPR;
  __shared__ float red[2][LPR > 64 ? LPR / 64 : 1][2];
  __shared__ float cols[FEW ? BLOCK / 32 * ln_columns<BLOCK>() * V : ROWS > 1 ? BLOCK * (V + 1) : 1];
  if (FEW && (int)blockIdx.x >= row_blocks)
    return layer_norm_columns<T, W, V, BLOCK>(dy, dstride, x, xstride, mean, rstd, dweight, dbias, (int)n, D, (int)blockIdx.x - row_blocks, cols);
  const int lane = threadIdx.x % LPR;
  const long step = (long)row_blocks * ROWS;
  // 128 registers at sixteen waves: the widest f32 rows have none left to keep where their pieces lie
  int c[NV], skip[NV];
  constexpr bool TIGHT = LPR == 1024 && NV == 4;
  auto places = [&]() {
    int end = D;
    asm volatile("" : "+s"(end));                               // (formed anew)
#pragma unroll
    for (int j = 0; j < NV; j++) ln_piece<V>(j * LPR + lane, end, c[j], skip[j], j < NV / 2);
  };
  RowPiece<W, V> wp[NV];
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    ln_piece<V>(j * LPR + lane, D, c[j], skip[j], j < NV / 2);
    if (w) wp[j] = row_get<W, V>(w + c[j]);
#pragma unroll
    for (int i = 0; i < V; i++) dw[j][i] = db[j][i] = 0.0f;
  }
  // the next row is on its way while this one is worked on, where the registers allow it
  constexpr bool AHEAD = LPR < 1024;
  RowPiece<T, V> pn[NV], dn[NV];
  float mun = 0.0f, rsn = 0.0f;
  auto fetch = [&](long r) {
#pragma unroll
    for (int j = 0; j < NV; j++) {
      pn[j] = row_get<T, V>(x + r * xstride + c[j]);
      dn[j] = row_get<T, V>(dy + r * dstride + c[j]);
    }
    mun = mean[r];
    rsn = rstd[r];
  };
  long r = (long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / LPR : 0);
  if (AHEAD && r < n) fetch(r);
  for (int turn = 0; r < n; r += step, turn ^= 1) {
    if (TIGHT) places();
    if (!AHEAD) fetch(r);
    RowPiece<T, V> p[NV], d[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      p[j] = pn[j];
      d[j] = dn[j];
    }
    const float mu = mun, rs = rsn;
    if (AHEAD && r + step < n) fetch(r + step);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float u = (float)d[j].e[i], h = ((float)p[j].e[i] - mu) * rs, g = w ? u * (float)wp[j].e[i] : u;
        if (!FEW) {
          db[j][i] += u;
          dw[j][i] += u * h;
        }
        s += i >= skip[j] ? g : 0.0f;
        q += i >= skip[j] ? g * h : 0.0f;
      }
    }
    row_sum2<LPR>(s, q, red[turn]);
    const float a = s * inv_d, b = q * inv_d;
    if (TIGHT) places();
#pragma unroll
    for (int j = 0; j < NV; j++) {
      row_pin(p[j]);                                            // g and xh are formed again from the 16-byte pieces: held over the sums
      row_pin(d[j]);                                            // they would take four times the registers
      float f[V];
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float u = (float)d[j].e[i], h = ((float)p[j].e[i] - mu) * rs, g = w ? u * (float)wp[j].e[i] : u;
        f[i] = (g - a - h * b) * rs;
      }
      if (skip[j] < V) row_put<T, V, false>(dx + r * D + c[j], f);
    }
  }
  if (FEW || !part) return;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (!(k ? dbias : dweight)) continue;                        // (that half is not read)
#pragma unroll
    for (int j = 0; j < NV; j++) {
      float(&acc)[V] = k ? db[j] : dw[j];
      if (ROWS > 1) {                                            // the workgroup's rows meet in LDS
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++) cols[threadIdx.x * (V + 1) + i] = acc[i];
        __syncthreads();
        if (threadIdx.x < LPR) {
#pragma unroll
          for (int t = 1; t < ROWS; t++)
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] += cols[(t * LPR + lane) * (V + 1) + i];
        }
      }
      if (threadIdx.x < LPR && skip[j] < V) row_put<float, V, false>(part + ((long)blockIdx.x * 2 + k) * D + c[j], acc);
    }
  }
}

// dw | db [2 D] from the workgroups' partial rows: COLS columns per workgroup, 1024 / COLS groups of lanes share the rows and meet through
// shuffles and LDS.  COLS = 16 up to 1024 columns, where 64 leave most of the chip idle (230400 x 128: the whole pass 39.4 -> 37.8 us);
// 64 beyond, whole 256-byte pieces (16384 x 4096: 4.8 us, with 16 columns 7.2).
template <typename W, int COLS>
__global__ __launch_bounds__(1024) void layer_norm_wgrad_kernel(const float* __restrict__ part, int parts, int D, W* __restrict__ dw,
                                                                W* __restrict__ db) {
  __shared__ float red[16][COLS];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int c = blockIdx.x * COLS + lane % COLS;
  const bool asked = c < 2 * D && (c < D ? dw : db);
  float s = 0.0f;
  if (asked) {
#pragma unroll 8
    for (int i = threadIdx.x / COLS; i < parts; i += 1024 / COLS) s += part[(long)i * 2 * D + c];
  }
#pragma unroll
  for (int o = COLS; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
  if (lane < COLS) red[wv][lane] = s;
  __syncthreads();
  if (threadIdx.x < COLS && asked) {
    s = red[0][lane];
#pragma unroll
    for (int i = 1; i < 16; i++) s += red[i][lane];
    if (c < D) dw[c] = (W)s;
    else db[c - D] = (W)s;
  }
}

// ---------------------------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------------------------
// Calls f(V, LPR, NV) with the elements of a piece, the lanes per row and the pieces per lane of a row of D elements.  V is 16 bytes, or one
// element where a row is shorter.  Up to 128 pieces a wave (or less) holds a row and no barrier is needed; beyond, 2 to 16 waves.  Two
// pieces per lane: 256 lanes of one piece take 47 us instead of 38 forward (32768 x 1500 bf16; backward the same 63), 256 lanes of four 55
// instead of 52 and 82 instead of 80 (8192 x 8192).  NV > 1 implies more than LPR * NV / 2 pieces: the first half of a lane's are whole.
template <int N>
struct LnInt { static constexpr int v = N; };

template <int V, typename F>
static void ln_shape(int D, F g) {
  const int pieces = (D + V - 1) / V;
  auto f = [&](auto lpr, auto nv) { g(LnInt<V>(), lpr, nv); };
  if (D < V) g(LnInt<1>(), LnInt<8>(), LnInt<1>());
  else if (pieces <= 8) f(LnInt<8>(), LnInt<1>());
  else if (pieces <= 16) f(LnInt<16>(), LnInt<1>());
  else if (pieces <= 32) f(LnInt<32>(), LnInt<1>());
  else if (pieces <= 64) f(LnInt<64>(), LnInt<1>());
  else if (pieces <= 128) f(LnInt<64>(), LnInt<2>());
  else if (pieces <= 256) f(LnInt<128>(), LnInt<2>());
  else if (pieces <= 512) f(LnInt<256>(), LnInt<2>());
  else if (pieces <= 1024) f(LnInt<512>(), LnInt<2>());
  else if (pieces <= 2048) f(LnInt<1024>(), LnInt<2>());
  else if constexpr (V == 4) f(LnInt<1024>(), LnInt<4>());
}

// calls f(element, weight element) for a pair of dtypes; false: not a pair that the kernels have
template <typename F>
static bool ln_types(int dtype, int wdtype, F f) {
  if (dtype == NS_F32 && wdtype == NS_F32) f(0.0f, 0.0f);
  else if (dtype == NS_F16 && wdtype == NS_F16) f((_Float16)0, (_Float16)0);
  else if (dtype == NS_F16 && wdtype == NS_F32) f((_Float16)0, 0.0f);
  else if (dtype == NS_BF16 && wdtype == NS_BF16) f((rw_bf16)0.0f, (rw_bf16)0.0f);
  else if (dtype == NS_BF16 && wdtype == NS_F32) f((rw_bf16)0.0f, 0.0f);
  else return false;
  return true;
}

// Most workgroups by shape: enough to fill the chip, few enough that weights are fetched (and, backward, a partial row pair is left) once per
// many rows.  Measured neighbours, us.  Forward: 512 columns bf16 (8192) 24.6, half / twice as many 24.3 / 26.6; 1500 (8192) 38.5, 39.0 /
// 39.5; 4096 (4096) 47, 51 / 47; 16384 (256) 57, twice / four times 59 / 64.  Backward: 128 f16 (768) 36.4, 512 / 1024 37.9 / 36.4; 1500
// bf16 (1024) 63, 768 / 1536 68 / 80; 4096 (512) 82, 256 / 768 100 / 87; 8192 (256) 80, 512 / 768 87 / 92; 16384 (256) 90, 512 / 768 101 / 116.
struct LnMost {
  int forward, backward;
};
static LnMost ln_most(int pieces) {
  if (pieces <= 128) return {8192, 768};      // up to a wave per row
  if (pieces <= 256) return {8192, 1024};
  if (pieces <= 512) return {4096, 512};
  if (pieces <= 1024) return {1024, 256};
  return {256, 256};
}

// rows up to which the backward pass is one launch without a workspace (an allocation and a launch less: 14 us instead of 18 a call where the
// host is what it waits for).  On the device, us, one launch | two: 512 rows of 128 bf16 5.8 | 6.3, of 771: 6.3 | 7.0, of 4096: 9.6 | 16.8;
// 1024 rows: 7.6 | 6.4, 11.8 | 8.3, 14.3 | 18.5
#define LN_FEW_ROWS 512
static int ln_blocks(long n, int D, int vec, bool back) {
  const int pieces = (D + vec - 1) / vec;
  const int per = pieces <= 8 ? 32 : pieces <= 16 ? 16 : pieces <= 32 ? 8 : pieces <= 128 ? 4 : 1;
  const int most = back ? ln_most(pieces).backward : ln_most(pieces).forward;
  const long want = (n + per - 1) / per;
  return (int)(want < most ? want : most);
}

extern "C" int ns_layer_norm_forward(const void* x, long x_stride, const void* weight, const void* bias, int wdtype, void* y, float* mean,
                                     float* rstd, int dtype, long n, int cols, float eps, void* stream) {
  NS_REQUIRE(n >= 0 && n <= (1L << 40) && cols >= 1 && cols <= LN_MAX_COLS && x_stride >= 0,
             "ns_layer_norm_forward: bad shape (n %ld, cols %d in 1 .. %d)", n, cols, LN_MAX_COLS);
  NS_REQUIRE(eps > 0.0f && eps < __builtin_inff(), "ns_layer_norm_forward: eps %g has to be positive and finite", (double)eps);
  NS_REQUIRE((mean == nullptr) == (rstd == nullptr), "ns_layer_norm_forward: mean and rstd come together");
  if (n == 0) return NS_OK;
  NS_REQUIRE(x && y, "ns_layer_norm_forward: null pointer");
  NS_REQUIRE(row_aligned(x, dtype) && row_aligned(y, dtype) && row_aligned(weight, wdtype) && row_aligned(bias, wdtype) &&
                 row_aligned(mean, NS_F32) && row_aligned(rstd, NS_F32),
             "ns_layer_norm_forward: a pointer is not aligned to its elements");
  const bool ok = ln_types(dtype, wdtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    ln_shape<row_vec<T>()>(cols, [&](auto vec, auto lpr, auto nv) {
      constexpr int V = decltype(vec)::v, L = decltype(lpr)::v, N = decltype(nv)::v;
      hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W, V, L, N>), dim3(ln_blocks(n, cols, row_vec<T>(), false)), dim3(ln_block<L>()), 0,
                         (hipStream_t)stream, (const T*)x, x_stride, (const W*)weight, (const W*)bias, (T*)y, mean, rstd, n, cols,
                         1.0f / (float)cols, eps);
    });
  });
  NS_REQUIRE(ok, "ns_layer_norm_forward: dtype %d / weight dtype %d: NS_F16, NS_BF16 or NS_F32, weights the same or NS_F32", dtype, wdtype);
  NS_CHECK_LAUNCH("layer_norm_fwd_kernel");
  return NS_OK;
}

extern "C" size_t ns_layer_norm_backward_workspace_bytes(long n, int cols, int dtype) {
  if (n <= LN_FEW_ROWS || cols < 1 || cols > LN_MAX_COLS) return 0;
  return (size_t)ln_blocks(n, cols, dtype == NS_F32 ? 4 : 8, true) * 2 * cols * 4;
}

extern "C" int ns_layer_norm_backward(const void* dy, long dy_stride, const void* x, long x_stride, const float* mean, const float* rstd,
                                      const void* weight, int wdtype, void* dx, void* dweight, void* dbias, int dtype, long n, int cols,
                                      void* ws, size_t ws_bytes, void* stream) {
  NS_REQUIRE(n >= 0 && n <= (1L << 40) && cols >= 1 && cols <= LN_MAX_COLS && x_stride >= 0 && dy_stride >= 0,
             "ns_layer_norm_backward: bad shape (n %ld, cols %d in 1 .. %d)", n, cols, LN_MAX_COLS);
  NS_REQUIRE(n == 0 || (dy && x && mean && rstd && dx), "ns_layer_norm_backward: null pointer");
  NS_REQUIRE((weight != nullptr) == (dweight != nullptr), "ns_layer_norm_backward: weight and dweight come together");
  const bool sums = dweight || dbias;
  const size_t need = sums ? ns_layer_norm_backward_workspace_bytes(n, cols, dtype) : 0;
  NS_REQUIRE(ws_bytes >= need && (ws || need == 0), "ns_layer_norm_backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
  NS_REQUIRE(row_aligned(dy, dtype) && row_aligned(x, dtype) && row_aligned(dx, dtype) && row_aligned(weight, wdtype) &&
                 row_aligned(dweight, wdtype) && row_aligned(dbias, wdtype) && row_aligned(mean, NS_F32) && row_aligned(rstd, NS_F32) &&
                 row_aligned(ws, NS_F32),
             "ns_layer_norm_backward: a pointer is not aligned to its elements");
  const int blocks = ln_blocks(n, cols, dtype == NS_F32 ? 4 : 8, true);
  const bool ok = ln_types(dtype, wdtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    const bool few = n <= LN_FEW_ROWS;
    if (n > 0 || (sums && few))
      ln_shape<row_vec<T>()>(cols, [&](auto vec, auto lpr, auto nv) {
        constexpr int V = decltype(vec)::v, L = decltype(lpr)::v, N = decltype(nv)::v, wide = ln_columns<ln_block<L>()>() * V;
        const int extra = sums && few ? (cols + wide - 1) / wide : 0;
        auto kernel = few ? layer_norm_bwd_kernel<T, W, V, L, N, true> : layer_norm_bwd_kernel<T, W, V, L, N, false>;
        hipLaunchKernelGGL(kernel, dim3(blocks + extra), dim3(ln_block<L>()), 0, (hipStream_t)stream, (const T*)dy, dy_stride, (const T*)x,
                           x_stride, mean, rstd, (const W*)weight, (T*)dx, sums ? (float*)ws : nullptr, (W*)dweight, (W*)dbias, n, cols,
                           1.0f / (float)cols, blocks);
      });
    if (sums && !few && cols <= 1024)
      hipLaunchKernelGGL((layer_norm_wgrad_kernel<W, 16>), dim3((2 * cols + 15) / 16), dim3(1024), 0, (hipStream_t)stream, (const float*)ws,
                         blocks, cols, (W*)dweight, (W*)dbias);
    else if (sums && !few)
      hipLaunchKernelGGL((layer_norm_wgrad_kernel<W, 64>), dim3((2 * cols + 63) / 64), dim3(1024), 0, (hipStream_t)stream, (const float*)ws,
                         blocks, cols, (W*)dweight, (W*)dbias);
  });
  NS_REQUIRE(ok, "ns_layer_norm_backward: dtype %d / weight dtype %d: NS_F16, NS_BF16 or NS_F32, weights the same or NS_F32", dtype, wdtype);
  NS_CHECK_LAUNCH("layer_norm_bwd_kernel");
  return NS_OK;
}
