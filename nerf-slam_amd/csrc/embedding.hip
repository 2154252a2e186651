// embedding.hip -- rows of a table looked up by id (a latent per keyframe, a vector per token) and the table's gradient.
//
//   forward    out[t] = round(scale * table[id_t])
//   gradient   grad[r] = round(scale * sum over t with id_t = r of dout[t])       (rows that no token names: 0)
// An id outside [0, rows) is a padded place: its output row is zero and its upstream gradient is not used (it may be read: the sums load
// every place of the sorted list, and what belongs to no row goes nowhere).
//
// The gradient is a sum over the tokens SORTED by id, without floating-point atomics: the order of every sum is fixed by the ids
// alone, so the same inputs give the same bits.  All sorts are stable.  Three forms, by sizes (times of one call on the device):
//   short list   n <= SMALL_MAX: one launch; a workgroup owns neighbouring rows of the table and picks their tokens out of the whole list
//                (embed_small_kernel; 3001 tokens of 771 f32, 1013 rows: 11 us)
//   few rows     up to FEW_ROWS rows of up to 16 lanes: two launches; a workgroup sorts and sums a tile of tokens, then the tiles' sums are
//                added per row (embed_tile_kernel, embed_rows_kernel; 262144 tokens of 32 f16, 512 rows: 14 us, 26 in the next form)
//   general      sort, sums over equal shares of the sorted list -- so that a row that a tenth of the tokens name costs no more than any
//                other --, join (50000 rows of bf16: 16384 tokens of 1024 40 us = 3.4 TB/s of its 135 MB, 65536 tokens of 1024
//                80 us = 2.9, of 2048 126 us = 3.7)
//     sort   n <= RANK_MAX: one launch, a token's place counted directly (embed_rank_kernel); longer: radix passes of up to 10 bits, one
//            launch each up to ONE_MAX tokens (embed_pass_kernel), beyond as histogram, prefix, scatter
//     sums   a group of lanes walks consecutive places and sums runs of equal ids in f32 registers (emb_sum_share); a run inside the
//            workgroup's share is final, one that crosses its ends leaves one f32 partial row per share (embed_sum_kernel)
//     join   the share in which a crossing run begins adds its partial rows in order (embed_join_kernel)
// The general form moves little more than dout and the gradient; beside them it is bound by the latency of its launches, each a chain of
// dependent loads (16384 tokens of 1024: sort 24 us with the gradient's zeros written beside it, sums 11, join 4 of the 40; 65536 tokens:
// sort 35 us in six launches, sums 31, join 4).
//
// Columns: a lane holds V of them, 16 bytes, or one where a row is shorter than 16 bytes.  The last piece of a row ends with the row, so
// where D is no multiple of V it overlaps the one before: both lanes form the same sums in the same order and store the same bits.
// Outputs are stored past the caches (lookup of 65536 tokens of 2048 bf16: 87 -> 59 us; the gradient hardly minds, 65536 tokens of 512 bf16 with
// 32000 f32 rows: 58 -> 56).
#include "rows.h"

// ---- short list ----
#define SMALL_MAX 4096       // tokens.  At 4096, 1000 rows: 8 us (32 columns) and 10 (1024) against 13 and 13 in the general form; all tokens
                             // of one row: 12 and 21 against 12 and 25
#define SMALL_ROWS 256       // most rows of the table per workgroup
#define SMALL_BLOCKS 256     // workgroups aimed at -- one round on the chip; 512: 3001 tokens 17 us instead of 11 --, and a quarter of what is
                             // allowed (beyond, the general form)
#define SMALL_LANES 4        // log2 of the most lanes per row: a row that takes all of 4096 tokens of 1024 bf16 costs 21 us, with 64 lanes 55
// ---- few rows ----
#define FEW_ROWS (MAX_BINS - 1)   // 1000 rows, 262144 tokens of 64 f16 in random order: 29 us against 33 in the general form
#define FEW_LANES 4          // log2 of the most lanes per row: what is best depends on the ids' order, which the host does not know.  At 4 (128
                             // f16 columns) 262144 tokens take 24 against 33 us in runs of 64 equal ids, 42 against 38 in random order; 32768
                             // tokens 13 against 22 and 21.5 against 23.  At 5 (256 columns) 131072 tokens would take 24 against 33 in runs,
                             // 52 against 35 in random order
#define FEW_TILES 1024       // 2^20 tokens of 32 f16: 45 against 71 us; bounds the workspace
#define FEW_WAVES 8          // per tile; 4 or 16: 14.3 or 14.6 us instead of 13.7 at 262144 tokens of 32
// ---- general (50000 rows of bf16 unless stated) ----
#define RANK_MAX 8192        // 256 columns: 6000 / 8192 tokens 17 / 20 us against 21 / 22.5 with radix passes, 16384 tokens 41 against 30.  8192
                             // tokens of 1024 columns: 37 against 33, as two passes write the gradient's 102 MB of zeros in two launches
#define ONE_MAX 16384        // 16384 tokens, two passes: 30 us against 37 as three launches a pass (256 columns), 40 against 47 (1024); 32768
                             // tokens of 256: 43 against 41, 20000 of 1024: 44.5 against 49.5
#define TILE 1024            // tokens per workgroup of a radix pass and of the few rows' form
#define MAX_BITS 10          // of a radix pass' digit
#define MAX_BINS (1 << MAX_BITS)
#define SUM_U 8              // rows that a lane has on their way; 16: 86 instead of 56 us at 65536 tokens of 512, 32000 rows (fewer waves fit); 4: 56
#define GROUP 8              // places of the sorted list per group of lanes, doubled (up to 128) while more than GROUP_WAVES waves are
#define GROUP_WAVES 2048     // at work.  1024 / 4096 / 8192 waves: 41 / 41 / 41 instead of 39.5 us at 16384 tokens of 1024, 53 / 50 / 53 instead of
                             // 49 at 100000 of 256, 56 / 60.5 / 67 instead of 56 at 65536 of 512, 32000 rows

template <typename I>
__device__ __forceinline__ unsigned emb_key(I id, unsigned rows) {
  return id >= 0 && id < (I)rows ? (unsigned)id : rows;    // rows: the key of a padded place, sorted behind every row
}

// ---------------------------------------------------------------------------------------------
// forward: (1 << ls) lanes per token, EMB_C pieces of the row per lane (blockIdx.y: the next ones).  One token per group of lanes: with
// several, 65536 tokens of 2048 bf16 took 79 .. 87 us instead of 59 = 5.6 TB/s of its 332 MB, the rate of a large copy.
// ---------------------------------------------------------------------------------------------
#define EMB_C 4
template <typename T, int V, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, long tstride, const I* __restrict__ ids,
                                                        T* __restrict__ out, long n, unsigned rows, int D, int ls, float scale) {
  const int lane = threadIdx.x & ((1 << ls) - 1);
  const long t = (long)blockIdx.x * (256 >> ls) + (threadIdx.x >> ls);
  if (t >= n) return;
  const unsigned key = emb_key(ids[t], rows);
  const bool live = key < rows;
  const T* row = table + (live ? (long)key * tstride : 0);
  const int p0 = (int)blockIdx.y * EMB_C * (V << ls), p1 = min(D, p0 + EMB_C * (V << ls));
  for (int p = p0 + lane * V; p < p1; p += V << ls) {
    const int c = min(p, D - V);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = 0.0f;
    if (live) {
      const RowPiece<T, V> v = row_get<T, V>(row + c);
#pragma unroll
      for (int i = 0; i < V; i++) f[i] = (float)v.e[i] * scale;
    }
    row_put<T, V, true>(out + t * D + c, f);
  }
}

// ---------------------------------------------------------------------------------------------
// Rows without tokens: every launch of the sort, a few workgroups bound by latency, also writes a part of the whole gradient with zeros
// (workgroups from `sort` on); the sums that follow write the rows that have tokens again.
// ---------------------------------------------------------------------------------------------
// FILL_BLOCKS workgroups at most: more stores in flight hold up the sort's loads, fewer do not get the zeros written meanwhile.  64 / 256 / 512
// of them: 50000 rows of 1024 bf16 (102 MB), 16384 tokens 39 / 42 / 41 instead of 39.5 us, 65536 tokens 84 / 80.5 / 81 instead of 80; of 2048
// (205 MB) 143 / 128 / 129 instead of 126; 300000 rows of 1024 f32 (1.2 GB), 16384 tokens 267 / 252 / 266 instead of 250, 65536 tokens 376 / 278 /
// 293 instead of 262.  (In the form before, the sums wrote the zeros: 46 us for the first.)
#define FILL_BYTES (1 << 14)     // per workgroup
#define FILL_BLOCKS 128
struct EmbFill {
  char* at;
  long bytes;      // of whole elements
  int sort;        // workgroups that sort
};

__device__ __forceinline__ void emb_fill(const EmbFill& f, int threads) {
  typedef int v4i __attribute__((ext_vector_type(4), aligned(2)));
  const long step = (long)((int)gridDim.x - f.sort) * threads * 16;
  for (long o = ((long)((int)blockIdx.x - f.sort) * threads + threadIdx.x) * 16; o < f.bytes; o += step) {
    if (o + 16 <= f.bytes) {
      __builtin_nontemporal_store(v4i{0, 0, 0, 0}, reinterpret_cast<v4i*>(f.at + o));
    } else {
      for (long i = o; i < f.bytes; i += 2) *reinterpret_cast<short*>(f.at + i) = 0;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sort, short lists: the place of token t is the number of tokens with a smaller key, or the same key and a smaller index: n^2 compares
// at two vector instructions.  A workgroup places RANK_TOKENS tokens; its 16 waves, and the parts of a wave, each compare them with their
// part of the list, which lies in LDS.
// ---------------------------------------------------------------------------------------------
#define RANK_WAVES 16
#define RANK_TOKENS 16       // = RANK_WAVES: wave w compares the workgroup's tokens with its w-th
template <typename I>
__global__ __launch_bounds__(64 * RANK_WAVES) void embed_rank_kernel(const I* __restrict__ ids, int n, unsigned rows,
                                                                     unsigned* __restrict__ keys, int* __restrict__ order, EmbFill fill) {
  if ((int)blockIdx.x >= fill.sort) return emb_fill(fill, 64 * RANK_WAVES);
  constexpr int THREADS = 64 * RANK_WAVES, PARTS = THREADS / RANK_TOKENS;
  __shared__ __align__(16) unsigned k[RANK_MAX];
  __shared__ int cnt[RANK_WAVES][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int n4 = (n + 3) & ~3;
  I id[RANK_MAX / THREADS];
#pragma unroll
  for (int u = 0; u < RANK_MAX / THREADS; u++) id[u] = u * THREADS < n ? ids[min(u * THREADS + tid, n - 1)] : (I)0;
#pragma unroll
  for (int u = 0; u < RANK_MAX / THREADS; u++) {
    const int i = u * THREADS + tid;
    if (i < n4) k[i] = i < n ? emb_key(id[u], rows) : 0xffffffffu;       // (sorted behind all)
  }
  __syncthreads();
  const int b0 = blockIdx.x * RANK_TOKENS, me = lane % RANK_TOKENS, t = b0 + me;
  const unsigned key = t < n ? k[t] : 0u;
  const int per = ((n4 / 4 + PARTS - 1) / PARTS) * 4;
  const int lo = min((tid / RANK_TOKENS) * per, n4), hi = min(lo + per, n4);
  unsigned c = 0;
#pragma unroll 4
  for (int i = lo; i < min(hi, b0); i += 4) {                     // before the workgroup's tokens: ties count
    const uint4 q = *reinterpret_cast<const uint4*>(&k[i]);
    c += (q.x <= key) + (q.y <= key) + (q.z <= key) + (q.w <= key);
  }
#pragma unroll 4
  for (int i = max(lo, b0 + RANK_TOKENS); i < hi; i += 4) {       // behind them: ties do not count
    const uint4 q = *reinterpret_cast<const uint4*>(&k[i]);
    c += (q.x < key) + (q.y < key) + (q.z < key) + (q.w < key);
  }
  {                                                               // among them: ties with a smaller index count
    const unsigned q = (unsigned)__builtin_amdgcn_readlane((int)key, w);
    c += lane < RANK_TOKENS && b0 + w < n && (q < key || (q == key && w < me));
  }
  cnt[w][lane] = (int)c;
  __syncthreads();
  if (w == 0) {
    int p = 0;
#pragma unroll
    for (int i = 0; i < RANK_WAVES; i++) p += cnt[i][lane];
#pragma unroll
    for (int o = RANK_TOKENS; o < 64; o <<= 1) p += __shfl_xor(p, o, 64);
    if (lane < RANK_TOKENS && t < n) {
      keys[p] = key;
      order[p] = t;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sort, long lists: stable radix passes from the low digit up.  keys_in == nullptr: the first pass reads the ids.
// ---------------------------------------------------------------------------------------------
template <typename I>
__device__ __forceinline__ unsigned emb_key_at(const I* __restrict__ ids, const unsigned* __restrict__ keys_in, long t, unsigned rows) {
  return keys_in ? keys_in[t] : emb_key(ids[t], rows);
}

// Digits are counted in COPIES copies of the counters, by lane: where the same id fills a wave, its LDS atomics queue up a quarter as long.
#define COPIES 4
template <typename I>
__global__ __launch_bounds__(256) void embed_hist_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys_in, long n,
                                                         unsigned rows, int shift, int bins, int used,
                                                         int* __restrict__ hist, EmbFill fill) {
  if ((int)blockIdx.x >= fill.sort) return emb_fill(fill, 256);
  __shared__ int h[COPIES * MAX_BINS];
  const int tid = threadIdx.x, copy = tid & (COPIES - 1);
  for (int i = tid; i < COPIES * bins; i += 256) h[i] = 0;
  __syncthreads();
  const long t0 = (long)blockIdx.x * TILE + tid;
  unsigned key[TILE / 256];
#pragma unroll
  for (int i = 0; i < TILE / 256; i++) key[i] = emb_key_at(ids, keys_in, min(t0 + i * 256, n - 1), rows);
#pragma unroll
  for (int i = 0; i < TILE / 256; i++)
    if (t0 + i * 256 < n) atomicAdd(&h[((key[i] >> shift) & (bins - 1)) * COPIES + copy], 1);
  __syncthreads();
  for (int i = tid; i < used; i += 256) {
    int c = 0;
#pragma unroll
    for (int k = 0; k < COPIES; k++) c += h[i * COPIES + k];
    hist[(long)blockIdx.x * used + i] = c;
  }
}

// hist[tile][digit] -> tokens of that digit in earlier tiles; total[digit].  64 digits per workgroup (one per lane), the tiles shared by
// its 16 waves, 16 loads in flight each.
__global__ __launch_bounds__(1024) void embed_prefix_kernel(int* __restrict__ hist, int tiles, int bins, int* __restrict__ total,
                                                            EmbFill fill) {
  if ((int)blockIdx.x >= fill.sort) return emb_fill(fill, 1024);
  __shared__ int sums[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int d = blockIdx.x * 64 + lane;
  int run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    int v[16], mine = 0;
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int t = t0 + w * 16 + u;
      v[u] = t < tiles && d < bins ? hist[(long)t * bins + d] : 0;
      mine += v[u];
    }
    sums[w][lane] = mine;
    __syncthreads();
    int at = run;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      at += i < w ? sums[i][lane] : 0;
      run += sums[i][lane];
    }
#pragma unroll
    for (int u = 0; u < 16; u++) {
      const int t = t0 + w * 16 + u;
      if (t < tiles && d < bins) hist[(long)t * bins + d] = at;
      at += v[u];
    }
    __syncthreads();
  }
  if (w == 0 && d < bins) total[d] = run;
}

// lanes of a wave whose digit is this lane's, one ballot per bit
__device__ __forceinline__ unsigned long long emb_same_digit(int d, int bits, bool in) {
  unsigned long long same = __ballot(in);
  for (int b = 0; b < bits; b++) {
    const unsigned long long m = __ballot((d >> b) & 1);
    same &= (d >> b) & 1 ? m : ~m;
  }
  return same;
}

// A wave places a quarter of the tile in order, 64 tokens at a time: lanes with the same digit find each other with one ballot per
// bit, and the wave's own counter of the digit moves on by their number.
template <typename I>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys_in,
                                                            const int* __restrict__ order_in, long n, unsigned rows, int shift,
                                                            int bits, int used, const int* __restrict__ hist,
                                                            const int* __restrict__ total, unsigned* __restrict__ keys_out,
                                                            int* __restrict__ order_out, EmbFill fill) {
  if ((int)blockIdx.x >= fill.sort) return emb_fill(fill, 256);
  __shared__ int off[4][MAX_BINS];
  __shared__ int part[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int bins = 1 << bits;
  const long t0 = (long)blockIdx.x * TILE + w * (TILE / 4);
  constexpr int STEPS = TILE / 256, PER = MAX_BINS / 256;
  // all loads first
  unsigned key[STEPS];
  int from[STEPS], tot[PER], before_tile[PER];
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const long t = min(t0 + s * 64 + lane, n - 1);
    key[s] = emb_key_at(ids, keys_in, t, rows);
    from[s] = order_in ? order_in[t] : (int)t;
  }
  // (thread: PER neighbouring digits)
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int d = tid * PER + i;
    tot[i] = d < used ? total[d] : 0;
    before_tile[i] = d < used ? hist[(long)blockIdx.x * used + d] : 0;
  }
  for (int i = tid; i < 4 * bins; i += 256) off[i >> bits][i & (bins - 1)] = 0;
  // first place of every digit: prefix of the totals
  int sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) sum += tot[i];
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int from = __shfl_up(upto, o, 64);
    upto += lane >= o ? from : 0;
  }
  if (lane == 63) part[w] = upto;
  __syncthreads();
  unsigned long long same[STEPS];                             // lanes with the same digit in each step
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const bool in = t0 + s * 64 + lane < n;
    const int d = (key[s] >> shift) & (bins - 1);
    same[s] = emb_same_digit(d, bits, in);
    if (in && (same[s] & ((1ull << lane) - 1)) == 0) off[w][d] += __popcll(same[s]);      // (the first of them; one wave, in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  int base = upto - sum;
#pragma unroll
  for (int i = 0; i < 3; i++) base += i < w ? part[i] : 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int d = tid * PER + i;
    if (d < used) {
      int p = base + before_tile[i];
      base += tot[i];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int c = off[q][d];
        off[q][d] = p;
        p += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const long t = t0 + s * 64 + lane;
    const bool in = t < n;
    const int d = (key[s] >> shift) & (bins - 1);
    const int before = __popcll(same[s] & ((1ull << lane) - 1));
    const int p = in ? off[w][d] : 0;                     // (read by every lane before the first of them moves it on: one wave, in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) off[w][d] = p + __popcll(same[s]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      keys_out[p + before] = key[s];
      order_out[p + before] = from[s];
    }
  }
}

// A pass in ONE launch, for lists that a workgroup can read whole: every workgroup counts the digits of the whole list and of what
// lies before its tile by itself (n / 1024 loads per thread from the L2) instead of waiting for two launches that do it once.
#define ONE_WAVES (TILE / 64)
#define ONE_COPIES 2
template <typename I>
__global__ __launch_bounds__(TILE) void embed_pass_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys_in,
                                                          const int* __restrict__ order_in, int n, unsigned rows, int shift, int bits,
                                                          unsigned* __restrict__ keys_out, int* __restrict__ order_out, EmbFill fill) {
  if ((int)blockIdx.x >= fill.sort) return emb_fill(fill, TILE);
  extern __shared__ int lds[];       // [bins][ONE_COPIES] before the tile, [bins][ONE_COPIES] from it on, [waves][bins] 16 bit of each wave
  __shared__ int part[ONE_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, copy = tid & (ONE_COPIES - 1);
  const int bins = 1 << bits, t0 = (int)blockIdx.x * TILE;
  int* cnt = lds;
  unsigned short* off = reinterpret_cast<unsigned short*>(lds + 2 * ONE_COPIES * bins);    // (places below ONE_MAX)
  const int t = t0 + tid;
  const bool in = t < n;
  constexpr int U = ONE_MAX / TILE;
  unsigned k[U];                                           // the whole list, loads first
#pragma unroll
  for (int u = 0; u < U; u++) k[u] = u * TILE < n ? emb_key_at(ids, keys_in, min(u * TILE + tid, n - 1), rows) : 0u;
  const unsigned key = emb_key_at(ids, keys_in, min(t, n - 1), rows);
  const int from = order_in ? order_in[min(t, n - 1)] : t;
  for (int i = tid; i < (2 * ONE_COPIES + ONE_WAVES / 2) * bins; i += TILE) lds[i] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; u++)
    if (u * TILE + tid < n) atomicAdd(&cnt[((u * TILE < t0 ? 0 : bins) + ((k[u] >> shift) & (bins - 1))) * ONE_COPIES + copy], 1);
  const int d = (key >> shift) & (bins - 1);
  const unsigned long long same = emb_same_digit(d, bits, in);
  const int before = __popcll(same & ((1ull << lane) - 1));
  if (in && before == 0) off[w * bins + d] = (unsigned short)__popcll(same);
  __syncthreads();
  // first place of every digit (at most one per thread), then of every wave's tokens of it
  int prior = 0, mine = 0;
  if (tid < bins) {
#pragma unroll
    for (int k = 0; k < ONE_COPIES; k++) {
      prior += cnt[tid * ONE_COPIES + k];
      mine += cnt[(bins + tid) * ONE_COPIES + k];
    }
    mine += prior;
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int from = __shfl_up(upto, o, 64);
    upto += lane >= o ? from : 0;
  }
  if (lane == 63) part[w] = upto;
  __syncthreads();
  if (tid < bins) {
    int at = upto - mine + prior;
#pragma unroll
    for (int i = 0; i < ONE_WAVES; i++) at += i < w ? part[i] : 0;
    int c[ONE_WAVES];
#pragma unroll
    for (int i = 0; i < ONE_WAVES; i++) c[i] = off[i * bins + tid];
#pragma unroll
    for (int i = 0; i < ONE_WAVES; i++) {
      off[i * bins + tid] = (unsigned short)at;
      at += c[i];
    }
  }
  __syncthreads();
  if (in) {
    const int p = off[w * bins + d] + before;
    keys_out[p] = key;
    order_out[p] = from;
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the sorted list
// ---------------------------------------------------------------------------------------------
// first place in [lo, hi) whose key is not below `key`, for a wave (uniform arguments): 64 probes a step, so three dependent loads where
// halving takes eighteen
__device__ __forceinline__ int emb_lower_bound_wave(const unsigned* __restrict__ keys, int lo, int hi, unsigned key) {
  const int lane = threadIdx.x & 63;
  while (lo < hi) {
    const int step = (int)(((unsigned)(hi - lo) + 63u) / 64u);
    const long at = lo + (long)lane * step;
    const int below = __popcll(__ballot(at < hi && keys[at < hi ? at : lo] < key));
    if (below == 0) return lo;
    const long last = lo + (long)(below - 1) * step;       // the last probe below the key
    lo = (int)last + 1;
    hi = (int)min((long)hi, last + step);
  }
  return lo;
}

// The sums of one workgroup over its share of a sorted list of n places: groups of 1 << ls lanes take `group` places each from `base` on and
// sum runs of equal keys in registers; runs that cross groups meet through shuffles and LDS.  key(p), token(p): the list; `from`: dout at
// the lane's columns.  done(key, sum): a run that lies inside the share; enter(sum), leave(sum): the part of the run that enters the
// share, of the one that leaves it.
template <typename T, int V, int WAVES, typename Key, typename Token, typename Done, typename Enter, typename Leave>
__device__ __forceinline__ void emb_sum_share(const T* __restrict__ from, long dstride, long base, int n, unsigned rows, int ls, int group,
                                              Key key, Token token, Done done, Enter enter, Leave leave) {
  const int tid = threadIdx.x, lane = tid & ((1 << ls) - 1);
  __shared__ float met[WAVES][64][V + 1];                        // per wave: the run that was open where its first group begins
  __shared__ bool on[WAVES];                                   // ... and whether it is still open where the wave ends
  const int gi = tid >> ls;
  const long p0l = base + (long)gi * group;
  const int p0 = (int)min(p0l, (long)n), p1 = min(p0 + group, n);
  unsigned cur = p0 < p1 ? key(p0) : rows;
  bool head = p0 > 0 && p0 < p1 && key(p0 - 1) == cur;
  const bool open = p0 < p1 && p1 < n && key(p1) == key(p1 - 1);
  const bool entered = head && cur < rows;                    // by a run that began before
  bool through = false, leaves = false;                        // that run goes on behind the group; another one does
  float in[V], acc[V];                                         // the sum of that run here; of the current run
#pragma unroll
  for (int i = 0; i < V; i++) in[i] = acc[i] = 0.0f;
  // SUM_U rows on their way at a time, and the next ones' places (padded places' rows are read like others: their sum goes nowhere)
  constexpr int U = SUM_U;
  unsigned kn[U];
  int next[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int p = max(min(p0 + u, p1 - 1), 0);
    kn[u] = p0 < p1 ? key(p) : rows;
    next[u] = p0 < p1 ? token(p) : 0;
  }
  for (int b = p0; b < p1; b += U) {
    unsigned k[U];
    RowPiece<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      k[u] = kn[u];
      v[u] = row_get<T, V>(from + (long)next[u] * dstride);
    }
    if (b + U < p1) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = min(b + U + u, p1 - 1);
        kn[u] = key(p);
        next[u] = token(p);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (b + u >= p1) break;
      if (k[u] != cur) {                                       // a run ends inside the group
        if (head) {
#pragma unroll
          for (int i = 0; i < V; i++) in[i] = acc[i];
        } else {
          done(cur, acc);
        }
        head = false;
        cur = k[u];
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] += (float)v[u].e[i];
    }
  }
  if (cur < rows) {                                            // (padded places, and groups behind the list: nothing)
    if (head) {
      through = open;
#pragma unroll
      for (int i = 0; i < V; i++) in[i] = acc[i];
    } else if (open) {
      leaves = true;
    } else {
      done(cur, acc);
    }
  }
  // what follows in the wave: in = sum of the entering run from this group to its end or the wave's, doubling the reach step by step
  const int wl = tid & 63, w = tid >> 6, wide = 1 << ls;
  for (int o = wide; o < 64; o <<= 1) {
    const bool more = through && wl + o < 64;
    const bool beyond = __shfl_down((int)through, o, 64) != 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float f = __shfl_down(in[i], o, 64);
      in[i] += more ? f : 0.0f;
    }
    through = more ? beyond : through;
  }
  if (wl < wide) {
#pragma unroll
    for (int i = 0; i < V; i++) met[w][wl][i] = in[i];
    if (wl == 0) on[w] = through;
  }
  if (__ballot(leaves)) {                                      // (a leaving run takes what the next group of the wave was entered by)
    const bool last = wl + wide >= 64;
    const bool goes = __shfl_down((int)through, wide, 64) != 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float f = __shfl_down(in[i], wide, 64);
      acc[i] += last ? 0.0f : f;
    }
    through = last || goes;                                    // (of the leaving run from here on)
  }
  __syncthreads();
  if (gi == 0 && entered) {                                    // the run that enters the share
    for (int j = 1; j < WAVES && on[j - 1]; j++)
#pragma unroll
      for (int i = 0; i < V; i++) in[i] += met[j][wl][i];
    enter(in);
  }
  if (leaves) {
    for (int j = w + 1; j < WAVES && through; j++) {
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] += met[j][lane][i];
      through = on[j];
    }
    if (through) {
      leave(acc);
    } else {
      done(cur, acc);
    }
  }
}

// grid: shares x pieces of the columns, the pieces of one share next to each other, so that the rows of dout are read whole at about the
// same time.  A share is what a workgroup sums: `group`
// places per group of lanes, (256 >> ls) groups.  The groups sum their runs in registers and meet in LDS, so that only the run that
// enters the share and the one that leaves it become partial rows: part [shares][2][D], row 0 entered, row 1 begins here and leaves.
template <typename T, int V, typename G>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T* __restrict__ dout, long dstride, const unsigned* __restrict__ keys,
                                                        const int* __restrict__ order, int n, unsigned rows, int D, int ls, int group,
                                                        int pieces, float scale, G* __restrict__ grad,
                                                        float* __restrict__ part) {
  const int tid = threadIdx.x, block = (int)(blockIdx.x / (unsigned)pieces), lane = tid & ((1 << ls) - 1);
  const int first = (int)(blockIdx.x - (unsigned)block * pieces) * (V << ls) + lane * V, c = min(first, D - V);
  const bool col = first < D;
  auto store = [&](unsigned r, float* acc) {
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] *= scale;
    if (col) row_put<G, V, true>(grad + (long)r * D + c, acc);
  };
  auto keep = [&](float* acc, int k) {
    if (col) row_put<float, V, false>(part + ((long)block * 2 + k) * D + c, acc);
  };
  emb_sum_share<T, V, 4>(
      dout + c, dstride, (long)block * group * (256 >> ls), n, rows, ls, group, [&](int p) { return keys[p]; },
      [&](int p) { return order[p]; }, store, [&](float* acc) { keep(acc, 0); }, [&](float* acc) { keep(acc, 1); });
}

// grid (`each` shares each, pieces of the columns): a run that crosses the end of the share in which it begins is finished here.
// Its partial rows are added by sub-groups of lanes, each every (256 >> ls)-th of them, and the sub-groups are joined in order through LDS.
template <typename G, int V>
__global__ __launch_bounds__(256) void embed_join_kernel(const unsigned* __restrict__ keys, int n, unsigned rows, int D, int ls,
                                                         int share, float scale, G* __restrict__ grad, const float* __restrict__ part,
                                                         int each) {
  __shared__ float red[256][V + 1];
  const int tid = threadIdx.x, sub = tid >> ls, subs = 256 >> ls;
  const int first = (int)blockIdx.y * (V << ls) + (tid & ((1 << ls) - 1)) * V, c = min(first, D - V);
  const bool col = first < D;
  bool mine = false;                                           // every wave finds the same shares
  {
    const int i = tid & 63;
    const long p0 = ((long)blockIdx.x * each + i) * share, p1 = p0 + share;
    if (i < each && p1 < n) {
      const unsigned cur = keys[p1 - 1];
      mine = cur < rows && keys[p1] == cur && (p0 == 0 || keys[p0 - 1] != cur);
    }
  }
  unsigned long long todo = __ballot(mine);
  while (todo) {
    const int g = (int)blockIdx.x * each + __ffsll(todo) - 1;
    todo &= todo - 1;
    const int p1 = (g + 1) * share;
    const unsigned cur = keys[p1];
    // partial rows: [g][1], [g + 1][0], [g + 2][0], ...: one for every share that the run enters.  64 shares' beginnings are looked at;
    // a longer run is searched for
    const long begin = p1 + ((long)(tid & 63) + 1) * share;
    const unsigned long long enters = __ballot(begin < n && keys[begin < n ? begin : p1] == cur);
    int m = 2 + __popcll(enters);
    if (enters == ~0ull) m = (emb_lower_bound_wave(keys, p1, n, cur + 1u) - 1) / share - g + 1;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    if (col) {
#pragma unroll 8
      for (int i = sub; i < m; i += subs) {
        const RowPiece<float, V> v = row_get<float, V>(part + ((long)(g + i) * 2 + (i == 0 ? 1 : 0)) * D + c);
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] += v.e[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; e++) red[tid][e] = acc[e];
    __syncthreads();
    if (sub == 0 && col) {
      for (int s = 1; s < min(subs, m); s++)
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] += red[(s << ls) + tid][e];
#pragma unroll
      for (int e = 0; e < V; e++) acc[e] *= scale;
      row_put<G, V, true>(grad + (long)cur * D + c, acc);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Few, narrow rows and many tokens (the samples of a training step and their keyframes' latents): two launches instead of five.  A
// workgroup sorts its TILE tokens in LDS and leaves one sum per row that occurs among them, part [rows][tiles][D], and a bit for it in
// touched [tiles][32]; then a workgroup per row adds the tiles' sums in order.
// ---------------------------------------------------------------------------------------------
template <typename T, int V, typename I>
__global__ __launch_bounds__(64 * FEW_WAVES) void embed_tile_kernel(const T* __restrict__ dout, long dstride, const I* __restrict__ ids, int n,
                                                         unsigned rows, int D, int ls, int tiles, float* __restrict__ part,
                                                         unsigned* __restrict__ touched) {
  __shared__ __align__(4) unsigned short off[FEW_WAVES][MAX_BINS];
  __shared__ unsigned short key_of[TILE], token_of[TILE];
  __shared__ unsigned bits[MAX_BINS / 32];
  __shared__ int sums[FEW_WAVES];
  constexpr int THREADS = 64 * FEW_WAVES, STEPS = TILE / THREADS, PER = MAX_BINS / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int tile = blockIdx.x;
  const int t0 = tile * TILE, have = min(n - t0, TILE);
  unsigned key[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; s++) key[s] = emb_key(ids[t0 + min((w * STEPS + s) * 64 + lane, have - 1)], rows);
  for (int i = tid; i < FEW_WAVES * MAX_BINS / 2; i += THREADS) reinterpret_cast<unsigned*>(off)[i] = 0;
  if (tid < MAX_BINS / 32) bits[tid] = 0;
  __syncthreads();
  unsigned long long same[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const bool in = (w * STEPS + s) * 64 + lane < have;
    same[s] = emb_same_digit((int)key[s], MAX_BITS, in);
    if (in && (same[s] & ((1ull << lane) - 1)) == 0) off[w][key[s]] += (unsigned short)__popcll(same[s]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  int tot[PER], cnt[PER][FEW_WAVES], sum = 0;                                       // (thread: PER neighbouring rows)
  unsigned seen = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    tot[i] = 0;
#pragma unroll
    for (int q = 0; q < FEW_WAVES; q++) {
      cnt[i][q] = off[q][tid * PER + i];
      tot[i] += cnt[i][q];
    }
    seen |= tot[i] ? 1u << i : 0u;
    sum += tot[i];
  }
  if (seen) atomicOr(&bits[tid * PER / 32], seen << (tid * PER % 32));
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int from = __shfl_up(upto, o, 64);
    upto += lane >= o ? from : 0;
  }
  if (lane == 63) sums[w] = upto;
  __syncthreads();
  int at = upto - sum;
#pragma unroll
  for (int i = 0; i < FEW_WAVES - 1; i++) at += i < w ? sums[i] : 0;
#pragma unroll
  for (int i = 0; i < PER; i++)
#pragma unroll
    for (int q = 0; q < FEW_WAVES; q++) {
      off[q][tid * PER + i] = (unsigned short)at;
      at += cnt[i][q];
    }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const int t = (w * STEPS + s) * 64 + lane;
    const bool in = t < have;
    const int before = __popcll(same[s] & ((1ull << lane) - 1));
    const int p = in ? off[w][key[s]] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) off[w][key[s]] = (unsigned short)(p + __popcll(same[s]));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      key_of[p + before] = (unsigned short)key[s];
      token_of[p + before] = (unsigned short)t;
    }
  }
  __syncthreads();
  if (tid < MAX_BINS / 32) touched[(long)tile * (MAX_BINS / 32) + tid] = bits[tid];
  const int first = (tid & ((1 << ls) - 1)) * V, c = min(first, D - V);
  const bool col = first < D;
  auto store = [&](unsigned r, float* acc) {
    if (col) row_put<float, V, false>(part + ((long)r * tiles + tile) * D + c, acc);
  };
  // (nothing enters or leaves: the share is the whole list)
  emb_sum_share<T, V, FEW_WAVES>(
      dout + (long)t0 * dstride + c, dstride, 0, have, rows, ls, STEPS << ls, [&](int p) { return (unsigned)key_of[p]; },
      [&](int p) { return (int)token_of[p]; }, store, [](float*) {}, [](float*) {});
}

// one workgroup per row
template <typename G, int V>
__global__ __launch_bounds__(256) void embed_rows_kernel(const float* __restrict__ part, const unsigned* __restrict__ touched, int tiles,
                                                         int D, int ls, float scale, G* __restrict__ grad) {
  __shared__ float red[4][1 << FEW_LANES][V + 1];
  __shared__ bool named[4];
  const int tid = threadIdx.x, sub = tid >> ls, subs = 256 >> ls;
  const int row = blockIdx.x;
  const int first = (tid & ((1 << ls) - 1)) * V, c = min(first, D - V);
  const float* from = part + (long)row * tiles * D + c;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; i++) acc[i] = 0.0f;
  bool some = false;
  constexpr int U = 8;
  for (int t = sub; t < tiles; t += U * subs) {
    unsigned word[U];
#pragma unroll
    for (int u = 0; u < U; u++) word[u] = t + u * subs < tiles ? touched[(long)(t + u * subs) * (MAX_BINS / 32) + (row >> 5)] : 0u;
#pragma unroll
    for (int u = 0; u < U; u++)
      if ((word[u] >> (row & 31)) & 1) {
        const RowPiece<float, V> v = row_get<float, V>(from + (long)(t + u * subs) * D);
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += v.e[i];
        some = true;
      }
  }
  // the sub-groups of a wave meet through shuffles, the waves through LDS; a row without tokens is 0 whatever the scale
  const int wide = 1 << ls, w = tid >> 6, lane = tid & 63;
  for (int o = wide; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] += __shfl_xor(acc[i], o, 64);
  if (lane < wide) {
#pragma unroll
    for (int i = 0; i < V; i++) red[w][lane][i] = acc[i];
  }
  const bool any = __ballot(some) != 0;
  if (lane == 0) named[w] = any;
  __syncthreads();
  if (tid < wide && first < D) {
    const bool all = named[0] | named[1] | named[2] | named[3];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = all ? (red[0][tid][i] + red[1][tid][i] + red[2][tid][i] + red[3][tid][i]) * scale : 0.0f;
    row_put<G, V, true>(grad + (long)row * D + c, acc);
  }
}

// ---------------------------------------------------------------------------------------------
// Short lists: everything in one launch.  A workgroup owns `own` neighbouring rows of the table: it picks their tokens out of the whole list,
// sorts them in LDS, sums them and writes its rows, those without tokens too.  No workspace.
// grid: groups of rows x pieces of the columns
// ---------------------------------------------------------------------------------------------
#define SMALL_STEPS (SMALL_MAX / 1024)
template <typename T, int V, typename G, typename I>
__global__ __launch_bounds__(1024) void embed_small_kernel(const T* __restrict__ dout, long dstride, const I* __restrict__ ids, int n,
                                                           unsigned rows, int D, int ls, int pieces, int own, float scale,
                                                           G* __restrict__ grad) {
  __shared__ unsigned short off[16][SMALL_ROWS];
  __shared__ unsigned char key_of[SMALL_MAX];
  __shared__ unsigned short token_of[SMALL_MAX];
  __shared__ unsigned long long s_empty[SMALL_ROWS / 64];
  __shared__ int sums[SMALL_ROWS / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const unsigned block = blockIdx.x / (unsigned)pieces, r0 = block * own;
  // (a wave takes SMALL_STEPS x 64 neighbouring tokens)
  unsigned d[SMALL_STEPS];
#pragma unroll
  for (int s = 0; s < SMALL_STEPS; s++) {
    const int t = (w * SMALL_STEPS + s) * 64 + lane;
    const unsigned k = n > 0 ? emb_key(ids[min(t, n - 1)], rows) : rows;
    d[s] = t < n && k < rows ? k - r0 : 0xffffffffu;           // (rows below r0 wrap around)
  }
  for (int i = tid; i < 16 * SMALL_ROWS; i += 1024) off[i / SMALL_ROWS][i % SMALL_ROWS] = 0;
  __syncthreads();
  unsigned long long same[SMALL_STEPS];
#pragma unroll
  for (int s = 0; s < SMALL_STEPS; s++) {
    const bool in = d[s] < (unsigned)own;
    same[s] = 0;
    if (__ballot(in)) {
      same[s] = emb_same_digit((int)(d[s] & (SMALL_ROWS - 1)), 8, in);
      if (in && (same[s] & ((1ull << lane) - 1)) == 0) off[w][d[s]] += (unsigned short)__popcll(same[s]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  __syncthreads();
  int upto = 0, sum = 0;                                       // (thread: row)
  if (tid < SMALL_ROWS) {
#pragma unroll
    for (int q = 0; q < 16; q++) sum += off[q][tid];
    upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int from = __shfl_up(upto, o, 64);
      upto += lane >= o ? from : 0;
    }
    const unsigned long long empty = __ballot(sum == 0 && tid < own && r0 + tid < rows);
    if (lane == 0) s_empty[w] = empty;
    if (lane == 63) sums[w] = upto;
  }
  __syncthreads();
  int found = 0;
#pragma unroll
  for (int q = 0; q < SMALL_ROWS / 64; q++) found += sums[q];
  if (tid < SMALL_ROWS) {
    int at = upto - sum, c[16];
#pragma unroll
    for (int q = 0; q < SMALL_ROWS / 64; q++) at += q < w ? sums[q] : 0;
#pragma unroll
    for (int q = 0; q < 16; q++) c[q] = off[q][tid];
#pragma unroll
    for (int q = 0; q < 16; q++) {
      off[q][tid] = (unsigned short)at;
      at += c[q];
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < SMALL_STEPS; s++) {
    const bool in = d[s] < (unsigned)own;
    const int before = __popcll(same[s] & ((1ull << lane) - 1));
    const int p = in ? off[w][d[s]] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) off[w][d[s]] = (unsigned short)(p + __popcll(same[s]));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      key_of[p + before] = (unsigned char)d[s];
      token_of[p + before] = (unsigned short)((w * SMALL_STEPS + s) * 64 + lane);
    }
  }
  __syncthreads();
  const int first = (int)(blockIdx.x - block * pieces) * (V << ls) + (tid & ((1 << ls) - 1)) * V, c = min(first, D - V);
  const bool col = first < D;
  auto store = [&](unsigned r, float* acc) {
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] *= scale;
    if (col) row_put<G, V, true>(grad + ((long)r0 + r) * D + c, acc);
  };
  for (int r = tid >> ls; r < own; r += 1024 >> ls)
    if ((s_empty[r / 64] >> (r % 64)) & 1) {
      float z[V];
#pragma unroll
      for (int i = 0; i < V; i++) z[i] = 0.0f;
      if (col) row_put<G, V, true>(grad + ((long)r0 + r) * D + c, z);        // (0 whatever the scale)
    }
  const int groups = 1024 >> ls;
  if (found == 0) return;
  emb_sum_share<T, V, 16>(
      dout + c, dstride, 0, found, SMALL_ROWS, ls, (found + groups - 1) / groups, [&](int p) { return (unsigned)key_of[p]; },
      [&](int p) { return (int)token_of[p]; }, store, [](float*) {}, [](float*) {});
}

// ---------------------------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------------------------
// limits that keep every grid below 2^32 threads (up to 64 lanes per token, 16 per table row and piece of its columns; the sums' grid by
// EmbPlan::sums) and places in 32 bits
#define EMB_MAX_COLS 65536
#define EMB_MAX_TOKENS (1L << 25)
#define EMB_MAX_ROW_PIECES (1L << 27)     // rows x ceil(columns / 256) of a gradient
#define EMB_MAX_SUMS ((1L << 24) - 1)     // workgroups of 256 threads: only 2^25 tokens of more than 65280 f32 columns pass it

// small: group = rows per workgroup, shares = pieces of the columns
struct EmbPlan {
  bool small, ranked, few;
  int passes, bits, tiles, ls, group, shares;
  long sums;       // workgroups of embed_sum_kernel (general form)
  size_t keys[2], order[2], hist, total, part, touched, bytes;
};

static inline int emb_col_blocks(int cols, int vec, int ls) { return (cols + (vec << ls) - 1) / (vec << ls); }

static EmbPlan emb_plan(long n, long rows, int cols, int vec) {
  EmbPlan p = {};
  p.ls = row_lanes_log2(cols, vec);
  if (n <= SMALL_MAX) {
    // narrow pieces of the columns: a row that takes most of the tokens is still the work of several workgroups
    const int ls = p.ls < SMALL_LANES ? p.ls : SMALL_LANES, pieces = emb_col_blocks(cols, vec, ls);
    int own = 1;                                             // rows per workgroup
    while (own < SMALL_ROWS && (rows + own - 1) / own * pieces > SMALL_BLOCKS) own *= 2;
    if (n == 0 || (rows + own - 1) / own * pieces <= 4 * SMALL_BLOCKS) {
      p.small = true;
      p.ls = ls;
      p.group = own;
      p.shares = pieces;
      return p;
    }
  }
  p.ranked = n <= RANK_MAX;
  int need = 1;
  while (need < 32 && ((unsigned long)rows >> need) != 0) need++;         // keys 0 .. rows
  p.passes = p.ranked ? 0 : (need + MAX_BITS - 1) / MAX_BITS;
  p.bits = p.ranked ? 0 : (need + p.passes - 1) / p.passes;
  p.tiles = (int)((n + TILE - 1) / TILE);
  const long lanes = n * (((cols + vec - 1) / vec + (1 << p.ls) - 1) >> p.ls << p.ls);       // lanes at one place per group
  p.group = GROUP;
  while (p.group < 128 && lanes / p.group > 64L * GROUP_WAVES) p.group *= 2;
  const long share = (long)p.group * (256 >> p.ls);
  p.shares = (int)((n + share - 1) / share);
  size_t at = 0;
  auto take = [&at](size_t b) {
    const size_t was = at;
    at += (b + 255) & ~(size_t)255;
    return was;
  };
  p.few = !p.ranked && rows <= FEW_ROWS && p.ls <= FEW_LANES && p.tiles <= FEW_TILES;
  if (p.few) {
    p.touched = take((size_t)p.tiles * (MAX_BINS / 8));
    p.part = take((size_t)rows * p.tiles * cols * 4);
    p.bytes = at;
    return p;
  }
  for (int i = 0; i < 2; i++) {
    p.keys[i] = take(i == 0 || p.passes > 1 ? 4 * (size_t)n : 0);
    p.order[i] = take(i == 0 || p.passes > 1 ? 4 * (size_t)n : 0);
  }
  p.sums = (long)p.shares * emb_col_blocks(cols, vec, p.ls);
  p.hist = take(n <= ONE_MAX ? 0 : (size_t)p.tiles * (4u << p.bits));
  p.total = take(n <= ONE_MAX ? 0 : 4u << p.bits);
  p.part = take(p.shares > 1 ? (size_t)p.shares * 2 * cols * 4 : 0);
  p.bytes = at;
  return p;
}

template <int N>
struct EmbInt { static constexpr int v = N; };

// calls f(V): the elements that a lane holds of a row of D
template <typename T, typename F>
static void emb_pieces(int D, F f) {
  if (D >= row_vec<T>()) f(EmbInt<row_vec<T>()>());
  else f(EmbInt<1>());
}

// the same number, for a dtype of the C ABI
static int emb_vec(int dtype, int D) {
  const int v = dtype == NS_F32 ? 4 : 8;
  return D >= v ? v : 1;
}

static bool emb_fits(long n, long rows, int cols) {
  return n <= EMB_MAX_TOKENS && cols >= 1 && cols <= EMB_MAX_COLS && rows <= EMB_MAX_ROW_PIECES / ((cols + 255) / 256);
}

static inline bool emb_type(int dtype) { return dtype == NS_F16 || dtype == NS_BF16 || dtype == NS_F32; }

template <typename T, int V, typename I>
static void emb_forward(const void* table, long tstride, const void* ids, void* out, long n, long rows, int cols, float scale,
                        hipStream_t s) {
  const int ls = row_lanes_log2(cols, V);
  const int wide = EMB_C * (V << ls);
  hipLaunchKernelGGL((embed_fwd_kernel<T, V, I>), dim3((unsigned)((n + (256 >> ls) - 1) / (256 >> ls)), (cols + wide - 1) / wide), dim3(256), 0, s,
                     (const T*)table, tstride, (const I*)ids, (T*)out, n, (unsigned)rows, cols, ls, scale);
}

extern "C" int ns_embedding_forward(const void* table, long table_stride, const void* ids, int ids_are_64, void* out, int dtype,
                                    long n, long rows, int cols, float scale, void* stream) {
  NS_REQUIRE(n >= 0 && rows >= 0, "ns_embedding_forward: bad shape");
  NS_REQUIRE(emb_type(dtype), "ns_embedding_forward: dtype %d is not NS_F16, NS_BF16 or NS_F32", dtype);
  if (n == 0) return NS_OK;
  NS_REQUIRE(ids && out && (table || rows == 0), "ns_embedding_forward: null pointer");
  NS_REQUIRE(n <= EMB_MAX_TOKENS && rows <= 0x7fffffffL && cols >= 1 && cols <= EMB_MAX_COLS && table_stride >= 0,
             "ns_embedding_forward: bad shape (n %ld <= 2^25, rows %ld < 2^31, cols %d in 1 .. %d)", n, rows, cols, EMB_MAX_COLS);
  NS_REQUIRE(row_aligned(table, dtype) && row_aligned(out, dtype) && (uintptr_t)ids % (ids_are_64 ? 8 : 4) == 0,
             "ns_embedding_forward: a pointer is not aligned to its elements");
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    emb_pieces<T>(cols, [&](auto piece) {
      constexpr int V = decltype(piece)::v;
      if (ids_are_64) emb_forward<T, V, int64_t>(table, table_stride, ids, out, n, rows, cols, scale, s);
      else emb_forward<T, V, int32_t>(table, table_stride, ids, out, n, rows, cols, scale, s);
    });
  };
  if (dtype == NS_F16) go((_Float16)0);
  else if (dtype == NS_BF16) go((rw_bf16)0.0f);
  else go(0.0f);
  NS_CHECK_LAUNCH("embed_fwd_kernel");
  return NS_OK;
}

extern "C" size_t ns_embedding_backward_workspace_bytes(long n, long rows, int cols, int dtype) {
  if (n <= 0 || rows <= 0 || !emb_fits(n, rows, cols)) return 0;
  const EmbPlan p = emb_plan(n, rows, cols, emb_vec(dtype, cols));
  return p.sums <= EMB_MAX_SUMS ? p.bytes : 0;
}

template <typename I>
static void emb_sort(const EmbPlan& p, const I* ids, char* ws, int n, unsigned rows, void* grad, long grad_bytes, const unsigned** keys,
                     const int** order, hipStream_t s) {
  unsigned* k[2] = {(unsigned*)(ws + p.keys[0]), (unsigned*)(ws + p.keys[1])};
  int* o[2] = {(int*)(ws + p.order[0]), (int*)(ws + p.order[1])};
  // the gradient's zeros, in equal parts over the launches
  const int launches = p.ranked ? 1 : n <= ONE_MAX ? p.passes : 3 * p.passes;
  const long part = ((grad_bytes + launches - 1) / launches + 15) / 16 * 16;
  long filled = 0;
  EmbFill fill;
  auto grid = [&](int sort) {                                  // workgroups of a launch that sorts with `sort` of them; sets `fill`
    fill.at = (char*)grad + filled;
    fill.bytes = grad_bytes - filled < part ? grad_bytes - filled : part;
    fill.sort = sort;
    filled += fill.bytes;
    return dim3((unsigned)(sort + min((fill.bytes + FILL_BYTES - 1) / FILL_BYTES, (long)FILL_BLOCKS)));
  };
  if (p.ranked) {
    const dim3 g = grid((n + RANK_TOKENS - 1) / RANK_TOKENS);
    hipLaunchKernelGGL(embed_rank_kernel<I>, g, dim3(64 * RANK_WAVES), 0, s, ids, n, rows, k[0], o[0], fill);
    *keys = k[0];
    *order = o[0];
    return;
  }
  int* hist = (int*)(ws + p.hist);
  int* total = (int*)(ws + p.total);
  const int bins = 1 << p.bits;
  const unsigned* ki = nullptr;
  const int* oi = nullptr;
  for (int i = 0; i < p.passes; i++) {
    const int shift = i * p.bits;
    if (n <= ONE_MAX) {
      const dim3 g = grid(p.tiles);
      hipLaunchKernelGGL(embed_pass_kernel<I>, g, dim3(TILE), (2 * ONE_COPIES + ONE_WAVES / 2) * sizeof(int) << p.bits, s, ids, ki, oi, n,
                         rows, shift, p.bits, k[i & 1], o[i & 1], fill);
    } else {
      const int used = (int)min((unsigned)bins, (rows >> shift) + 1);        // digits that occur: the keys end at `rows`
      dim3 g = grid(p.tiles);
      hipLaunchKernelGGL(embed_hist_kernel<I>, g, dim3(256), 0, s, ids, ki, (long)n, rows, shift, bins, used, hist, fill);
      g = grid((used + 63) / 64);
      hipLaunchKernelGGL(embed_prefix_kernel, g, dim3(1024), 0, s, hist, p.tiles, used, total, fill);
      g = grid(p.tiles);
      hipLaunchKernelGGL(embed_scatter_kernel<I>, g, dim3(256), 0, s, ids, ki, oi, (long)n, rows, shift, p.bits, used, hist, total, k[i & 1],
                         o[i & 1], fill);
    }
    ki = k[i & 1];
    oi = o[i & 1];
  }
  *keys = ki;
  *order = oi;
}

template <typename T, int V, typename G, typename I>
static void emb_small(const EmbPlan& p, const T* dout, long dstride, const I* ids, int n, unsigned rows, int cols, float scale, G* grad,
                      hipStream_t s) {
  hipLaunchKernelGGL((embed_small_kernel<T, V, G, I>), dim3((rows + p.group - 1) / p.group * p.shares), dim3(1024), 0, s, dout, dstride, ids, n,
                     rows, cols, p.ls, p.shares, p.group, scale, grad);
}

template <typename T, int V, typename G, typename I>
static void emb_few(const EmbPlan& p, const T* dout, long dstride, const I* ids, int n, unsigned rows, int cols, float scale, G* grad,
                    char* ws, hipStream_t s) {
  float* part = (float*)(ws + p.part);
  unsigned* touched = (unsigned*)(ws + p.touched);
  hipLaunchKernelGGL((embed_tile_kernel<T, V, I>), dim3(p.tiles), dim3(64 * FEW_WAVES), 0, s, dout, dstride, ids, n, rows, cols, p.ls, p.tiles, part,
                     touched);
  hipLaunchKernelGGL((embed_rows_kernel<G, V>), dim3(rows), dim3(256), 0, s, part, touched, p.tiles, cols, p.ls, scale, grad);
}

template <typename T, int V, typename G>
static void emb_sums(const EmbPlan& p, const T* dout, long dstride, const unsigned* keys, const int* order, int n, unsigned rows,
                     int cols, float scale, G* grad, float* part, hipStream_t s) {
  const int col_blocks = emb_col_blocks(cols, V, p.ls), share = p.group * (256 >> p.ls);
  hipLaunchKernelGGL((embed_sum_kernel<T, V, G>), dim3((unsigned)p.shares * col_blocks), dim3(256), 0, s, dout, dstride, keys, order, n, rows,
                     cols, p.ls, p.group, col_blocks, scale, grad, part);
  if (p.shares > 1) {
    // one workgroup per share up to 1024 of them (in a skewed list most are the beginning of a crossing run, each a chain of loads);
    // beyond, a workgroup looks at up to 64
    const int each = p.shares > 64 * 1024 ? 64 : (p.shares + 1023) / 1024;
    hipLaunchKernelGGL((embed_join_kernel<G, V>), dim3((p.shares - 1 + each - 1) / each, col_blocks), dim3(256), 0, s, keys, n, rows, cols,
                       p.ls, share, scale, grad, part, each);
  }
}

extern "C" int ns_embedding_backward(const void* dout, long dout_stride, int dtype, const void* ids, int ids_are_64, void* grad,
                                     int grad_dtype, long n, long rows, int cols, float scale, void* ws, size_t ws_bytes,
                                     void* stream) {
  NS_REQUIRE(n >= 0 && rows >= 0, "ns_embedding_backward: bad shape");
  NS_REQUIRE(emb_type(dtype) && (grad_dtype == dtype || grad_dtype == NS_F32),
             "ns_embedding_backward: dtype %d / grad dtype %d: NS_F16, NS_BF16 or NS_F32, and the gradient that or NS_F32", dtype, grad_dtype);
  if (rows == 0) return NS_OK;
  NS_REQUIRE(emb_fits(n, rows, cols) && dout_stride >= 0,
             "ns_embedding_backward: bad shape (n %ld <= 2^25, cols %d in 1 .. %d, rows %ld x ceil(cols / 256) <= 2^27)", n, cols, EMB_MAX_COLS,
             rows);
  const EmbPlan p = emb_plan(n, rows, cols, emb_vec(dtype, cols));
  NS_REQUIRE(p.sums <= EMB_MAX_SUMS, "ns_embedding_backward: bad shape (n %ld of %d f32 columns: n <= 2^25 - 512 beyond 65280 columns)", n, cols);
  NS_REQUIRE(grad && (n == 0 || (dout && ids)) && (ws || p.bytes == 0), "ns_embedding_backward: null pointer");
  NS_REQUIRE(ws_bytes >= p.bytes, "ns_embedding_backward: workspace of %zu bytes, %zu needed", ws_bytes, p.bytes);
  NS_REQUIRE(((uintptr_t)ws % 16) == 0, "ns_embedding_backward: the workspace needs 16-byte alignment");
  NS_REQUIRE(row_aligned(dout, dtype) && row_aligned(grad, grad_dtype) && (uintptr_t)ids % (ids_are_64 ? 8 : 4) == 0,
             "ns_embedding_backward: a pointer is not aligned to its elements");
  hipStream_t s = (hipStream_t)stream;
  const unsigned* keys = nullptr;
  const int* order = nullptr;
  if (!p.small && !p.few) {
    const long bytes = rows * cols * (grad_dtype == NS_F32 ? 4 : 2);
    if (ids_are_64) emb_sort(p, (const int64_t*)ids, (char*)ws, (int)n, (unsigned)rows, grad, bytes, &keys, &order, s);
    else emb_sort(p, (const int32_t*)ids, (char*)ws, (int)n, (unsigned)rows, grad, bytes, &keys, &order, s);
    NS_CHECK_LAUNCH("embedding_backward: sort");
  }
  auto go = [&](auto t) {
    using T = decltype(t);
    float* part = (float*)((char*)ws + p.part);
    emb_pieces<T>(cols, [&](auto piece) {
      constexpr int V = decltype(piece)::v;
      auto small = [&](auto* g) {
        if (ids_are_64) emb_small<T, V>(p, (const T*)dout, dout_stride, (const int64_t*)ids, (int)n, (unsigned)rows, cols, scale, g, s);
        else emb_small<T, V>(p, (const T*)dout, dout_stride, (const int32_t*)ids, (int)n, (unsigned)rows, cols, scale, g, s);
      };
      auto few = [&](auto* g) {
        if (ids_are_64) emb_few<T, V>(p, (const T*)dout, dout_stride, (const int64_t*)ids, (int)n, (unsigned)rows, cols, scale, g, (char*)ws, s);
        else emb_few<T, V>(p, (const T*)dout, dout_stride, (const int32_t*)ids, (int)n, (unsigned)rows, cols, scale, g, (char*)ws, s);
      };
      if (p.small && grad_dtype == NS_F32)
        small((float*)grad);
      else if (p.small)
        small((T*)grad);
      else if (p.few && grad_dtype == NS_F32)
        few((float*)grad);
      else if (p.few)
        few((T*)grad);
      else if (grad_dtype == NS_F32)
        emb_sums<T, V, float>(p, (const T*)dout, dout_stride, keys, order, (int)n, (unsigned)rows, cols, scale, (float*)grad, part, s);
      else
        emb_sums<T, V, T>(p, (const T*)dout, dout_stride, keys, order, (int)n, (unsigned)rows, cols, scale, (T*)grad, part, s);
    });
  };
  if (dtype == NS_F16) go((_Float16)0);
  else if (dtype == NS_BF16) go((rw_bf16)0.0f);
  else go(0.0f);
  NS_CHECK_LAUNCH("embedding_backward: sums");
  return NS_OK;
}
