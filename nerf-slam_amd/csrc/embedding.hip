// embedding.hip -- rows of a table looked up by id (a latent per keyframe, a vector per token) and the table's gradient.
//
//   forward    out[t] = round(scale * table[id_t])
//   gradient   grad[r] = round(scale * sum over t with id_t = r of dout[t])       (rows that no token names: 0)
// An id outside [0, rows) is a padded place: its output row is zero and its upstream gradient is not read.
//
// The gradient is a sum over the tokens SORTED by id, without floating-point atomics: the order of every sum is fixed by the ids
// alone, so the same inputs give the same bits.  The sort is stable; its sums run over equal shares of the sorted list instead of
// over rows, so a row that a tenth of the tokens name costs no more than any other.
//   1. sort   n <= RANK_MAX: one launch, a token's place counted directly (embed_rank_kernel); longer: radix passes of up to 10 bits, one
//             launch each up to ONE_MAX tokens (embed_pass_kernel), beyond as histogram, prefix, scatter
//   2. sums   a group of lanes walks GROUP consecutive places and sums runs of equal ids in f32 registers; a run inside the share
//             is final, a run that crosses its ends leaves one f32 partial row per share
//   3. join   the share in which a crossing run begins adds its partial rows in order (embed_join_kernel)
#include "rows.h"

#define RANK_MAX 8192        // tokens whose places are counted directly
#define RANK_WAVES 16
#ifndef ONE_MAX
#define ONE_MAX 32768        // tokens up to which a radix pass is one launch
#endif
#define TILE 1024            // tokens per workgroup of a radix pass
#ifndef GROUP
#define GROUP 8              // places of the sorted list per group of lanes, doubled (to 128) while more than GROUP_WAVES waves are at work
#endif
#ifndef GROUP_WAVES
#define GROUP_WAVES 2048
#endif
#ifndef ZERO_ROWS
#define ZERO_ROWS 32         // table rows per wave that looks for rows without tokens
#endif
#ifndef EMB_U
#define EMB_U 4
#endif
#define MAX_BINS 1024

// ---------------------------------------------------------------------------------------------
// forward: lanes (1 << ls) per token, EMB_U tokens per group so that their id -> row round trips overlap
// ---------------------------------------------------------------------------------------------
template <typename I>
__device__ __forceinline__ unsigned emb_key(const I* __restrict__ ids, long t, unsigned rows) {
  const I v = ids[t];
  return v >= 0 && v < (I)rows ? (unsigned)v : rows;       // rows: the key of a padded place, sorted behind every row
}

template <typename T, typename I>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ table, long tstride, const I* __restrict__ ids,
                                                        T* __restrict__ out, long n, unsigned rows, int D, int ls, float scale) {
  constexpr int V = row_vec<T>();
  const int lane = threadIdx.x & ((1 << ls) - 1), grp = threadIdx.x >> ls, step = 256 >> ls;
  const long t0 = (long)blockIdx.x * (step * EMB_U) + grp;
  unsigned key[EMB_U];
#pragma unroll
  for (int u = 0; u < EMB_U; u++) {
    const long t = t0 + (long)u * step;
    key[u] = t < n ? emb_key(ids, t, rows) : rows;
  }
  for (int c = lane * V; c < D; c += V << ls) {
    RowPiece<T, V> v[EMB_U];
#pragma unroll
    for (int u = 0; u < EMB_U; u++) {
      if (key[u] < rows) {
        v[u] = row_load<T, V>(table + (long)key[u] * tstride, c, D);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[u].e[i] = (T)0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < EMB_U; u++) {
      const long t = t0 + (long)u * step;
      float f[V];
#pragma unroll
      for (int i = 0; i < V; i++) f[i] = key[u] < rows ? (float)v[u].e[i] * scale : 0.0f;   // (0 * scale: also where scale is inf)
      if (t < n) row_store<T, V, true>(out + t * D, c, D, f);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sort, short lists: the place of token t is the number of tokens with a smaller key, or the same key and a smaller index.  A
// workgroup places 64 tokens (one per lane); its 16 waves share the list, which lies in LDS.  n^2 compares at 2 vector
// instructions each.
// ---------------------------------------------------------------------------------------------
template <typename I>
__global__ __launch_bounds__(64 * RANK_WAVES) void embed_rank_kernel(const I* __restrict__ ids, int n, unsigned rows,
                                                                     unsigned* __restrict__ keys, int* __restrict__ order) {
  __shared__ __align__(16) unsigned k[RANK_MAX];
  __shared__ int cnt[RANK_WAVES][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int n4 = (n + 3) & ~3;
  for (int i = tid; i < n4; i += 64 * RANK_WAVES) k[i] = i < n ? emb_key(ids, i, rows) : 0xffffffffu;   // (sorted behind all)
  __syncthreads();
  const int b0 = blockIdx.x * 64, t = b0 + lane;
  const unsigned key = t < n ? k[t] : 0u;
  const int per = ((n4 / 4 + RANK_WAVES - 1) / RANK_WAVES) * 4;
  const int lo = min(w * per, n4), hi = min(lo + per, n4);
  int c = 0;
#pragma unroll 8
  for (int i = lo; i < min(hi, b0); i += 4) {                     // before the 64 tokens: ties count
    const uint4 q = *reinterpret_cast<const uint4*>(&k[i]);
    c += (q.x <= key) + (q.y <= key) + (q.z <= key) + (q.w <= key);
  }
#pragma unroll
  for (int u = 0; u < 64 / RANK_WAVES; u++) {                     // among them (their keys are the lanes' own): ties with a smaller
    const int i = w * (64 / RANK_WAVES) + u;                      // index count
    const unsigned q = (unsigned)__builtin_amdgcn_readlane((int)key, i);
    c += b0 + i < n && (q < key || (q == key && i < lane));
  }
#pragma unroll 8
  for (int i = max(lo, b0 + 64); i < hi; i += 4) {                // behind them: ties do not count
    const uint4 q = *reinterpret_cast<const uint4*>(&k[i]);
    c += (q.x < key) + (q.y < key) + (q.z < key) + (q.w < key);
  }
  cnt[w][lane] = c;
  __syncthreads();
  if (w == 0 && t < n) {
    int p = 0;
#pragma unroll
    for (int i = 0; i < RANK_WAVES; i++) p += cnt[i][lane];
    keys[p] = key;
    order[p] = t;
  }
}

// ---------------------------------------------------------------------------------------------
// sort, long lists: stable radix passes from the low digit up.  keys_in == nullptr: the first pass reads the ids.
// ---------------------------------------------------------------------------------------------
// Digits are counted in COPIES copies of the counters, by lane: where the same id fills a wave, its LDS atomics queue up a quarter as long.
#define COPIES 4
template <typename I>
__global__ __launch_bounds__(256) void embed_hist_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys_in, long n,
                                                         unsigned rows, int shift, int bins, int* __restrict__ hist) {
  __shared__ int h[COPIES * MAX_BINS];
  const int tid = threadIdx.x, copy = tid & (COPIES - 1);
  for (int i = tid; i < COPIES * bins; i += 256) h[i] = 0;
  __syncthreads();
  const long t0 = (long)blockIdx.x * TILE;
#pragma unroll
  for (int i = 0; i < TILE / 256; i++) {
    const long t = t0 + i * 256 + tid;
    if (t < n) {
      const unsigned key = keys_in ? keys_in[t] : emb_key(ids, t, rows);
      atomicAdd(&h[((key >> shift) & (bins - 1)) * COPIES + copy], 1);
    }
  }
  __syncthreads();
  for (int i = tid; i < bins; i += 256) {
    int c = 0;
#pragma unroll
    for (int k = 0; k < COPIES; k++) c += h[i * COPIES + k];
    hist[(long)blockIdx.x * bins + i] = c;
  }
}

// hist[tile][digit] -> tokens of that digit in earlier tiles; total[digit].  64 digits per workgroup (one per lane), the tiles shared by
// its 16 waves, 16 loads in flight each.
__global__ __launch_bounds__(1024) void embed_prefix_kernel(int* __restrict__ hist, int tiles, int bins, int* __restrict__ total) {
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
                                                            int bits, const int* __restrict__ hist, const int* __restrict__ total,
                                                            unsigned* __restrict__ keys_out, int* __restrict__ order_out) {
  __shared__ int off[4][MAX_BINS];
  __shared__ int part[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int bins = 1 << bits, per = (bins + 255) / 256;
  const long t0 = (long)blockIdx.x * TILE + w * (TILE / 4);
  constexpr int STEPS = TILE / 256;
  for (int i = tid; i < 4 * bins; i += 256) off[i >> bits][i & (bins - 1)] = 0;
  // first place of every digit: prefix of the totals (thread: `per` neighbouring digits)
  int sum = 0;
  for (int i = 0; i < per; i++) {
    const int d = tid * per + i;
    sum += d < bins ? total[d] : 0;
  }
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int from = __shfl_up(upto, o, 64);
    upto += lane >= o ? from : 0;
  }
  if (lane == 63) part[w] = upto;
  __syncthreads();
  unsigned key[STEPS];
  unsigned long long same[STEPS];                             // lanes with the same digit in each step
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    const long t = t0 + s * 64 + lane;
    key[s] = t < n ? (keys_in ? keys_in[t] : emb_key(ids, t, rows)) : 0u;
  }
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
  for (int i = 0; i < per; i++) {
    const int d = tid * per + i;
    if (d < bins) {
      int p = base + hist[(long)blockIdx.x * bins + d];
      base += total[d];
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
      order_out[p + before] = order_in ? order_in[t] : (int)t;
    }
  }
}

// A pass in ONE launch, for lists that a workgroup can read whole: every workgroup counts the digits of the whole list and of what
// lies before its tile by itself (n / 1024 loads per thread from the L2) instead of waiting for two launches that do it once.
#define ONE_WAVES (TILE / 64)
#ifndef ONE_COPIES
#define ONE_COPIES 2
#endif
template <typename I>
__global__ __launch_bounds__(TILE) void embed_pass_kernel(const I* __restrict__ ids, const unsigned* __restrict__ keys_in,
                                                          const int* __restrict__ order_in, int n, unsigned rows, int shift, int bits,
                                                          unsigned* __restrict__ keys_out, int* __restrict__ order_out) {
  extern __shared__ int lds[];       // [bins][ONE_COPIES] before the tile, [bins][ONE_COPIES] from it on, [waves][bins] 16 bit of each wave
  __shared__ int part[ONE_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, copy = tid & (ONE_COPIES - 1);
  const int bins = 1 << bits, t0 = (int)blockIdx.x * TILE;
  int* cnt = lds;
  unsigned short* off = reinterpret_cast<unsigned short*>(lds + 2 * ONE_COPIES * bins);    // (places below ONE_MAX)
  for (int i = tid; i < (2 * ONE_COPIES + ONE_WAVES / 2) * bins; i += TILE) lds[i] = 0;
  __syncthreads();
  unsigned key = 0;
#pragma unroll 4
  for (int b = 0; b < n; b += TILE) {
    const int i = b + tid;
    if (i < n) {
      const unsigned k = keys_in ? keys_in[i] : emb_key(ids, i, rows);
      const int d = (k >> shift) & (bins - 1);
      atomicAdd(&cnt[((b < t0 ? 0 : bins) + d) * ONE_COPIES + copy], 1);
      if (b == t0) key = k;
    }
  }
  const int t = t0 + tid;
  const bool in = t < n;
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
#pragma unroll
    for (int i = 0; i < ONE_WAVES; i++) {
      const int c = off[i * bins + tid];
      off[i * bins + tid] = (unsigned short)at;
      at += c;
    }
  }
  __syncthreads();
  if (in) {
    const int p = off[w * bins + d] + before;
    keys_out[p] = key;
    order_out[p] = order_in ? order_in[t] : t;
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the sorted list
// ---------------------------------------------------------------------------------------------
// first place in [lo, hi) whose key is not below `key`, for one lane
__device__ __forceinline__ int emb_lower_bound(const unsigned* __restrict__ keys, int lo, int hi, unsigned key) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (keys[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// the same for a whole wave (uniform arguments): 64 probes a step, so three dependent loads where the other takes eighteen
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

// grid (shares, then workgroups that write the rows without tokens; pieces of the columns).  A share is what a workgroup sums: `group`
// places per group of lanes, (256 >> ls) groups.  The groups sum their runs in registers and meet in LDS, so that only the run that
// enters the share and the one that leaves it become partial rows: part [shares][2][D], row 0 entered, row 1 begins here and leaves.
template <typename T, typename G>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T* __restrict__ dout, long dstride, const unsigned* __restrict__ keys,
                                                        const int* __restrict__ order, int n, unsigned rows, int D, int ls, int group,
                                                        int shares, float scale, G* __restrict__ grad, float* __restrict__ part) {
  constexpr int V = row_vec<T>();
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= shares) {                           // rows that no token names
    const int lane = tid & 63;
    const long r0 = ((long)((int)blockIdx.x - shares) * 4 + (tid >> 6)) * ZERO_ROWS;
    if (r0 >= (long)rows) return;
    const int lo = emb_lower_bound_wave(keys, 0, n, (unsigned)r0);
    const unsigned next = lo + lane < n ? keys[lo + lane] : 0xffffffffu;
    bool empty = false;
    if (__ballot(next >= (unsigned)r0 + ZERO_ROWS)) {          // 64 places show all tokens of these rows
#pragma unroll
      for (int i = 0; i < ZERO_ROWS; i++) {
        const bool none = __ballot(next == (unsigned)r0 + i) == 0;
        if (lane == i) empty = none && r0 + i < (long)rows;
      }
    } else if (lane < ZERO_ROWS && r0 + lane < (long)rows) {
      const unsigned r = (unsigned)(r0 + lane);
      const int p = emb_lower_bound(keys, lo, n, r);
      empty = p >= n || keys[p] != r;
    }
    unsigned long long m = __ballot(empty);
    const int c0 = (int)blockIdx.y * (V << ls), c1 = min(D, c0 + (V << ls));
    constexpr int VG = row_vec<G>();
    float z[VG];
#pragma unroll
    for (int i = 0; i < VG; i++) z[i] = 0.0f;
    while (m) {
      const int i = __ffsll(m) - 1;
      m &= m - 1;
      G* g = grad + (r0 + i) * (long)D;
      for (int c = c0 + lane * VG; c < c1; c += 64 * VG) row_store<G, VG, true>(g, c, c1, z);
    }
    return;
  }
  __shared__ float met[4][64][V + 1];                        // per wave: the run that was open where its first group begins
  __shared__ bool on[4];                                     // ... and whether it is still open where the wave ends
  const int lane = tid & ((1 << ls) - 1), gi = tid >> ls, groups = 256 >> ls;
  const int c = (int)blockIdx.y * (V << ls) + lane * V;
  const long p0l = ((long)blockIdx.x * groups + gi) * group;
  const int p0 = (int)min(p0l, (long)n), p1 = min(p0 + group, n);
  unsigned cur = p0 < p1 ? keys[p0] : rows;
  bool head = p0 > 0 && p0 < p1 && keys[p0 - 1] == cur;
  const bool open = p0 < p1 && p1 < n && keys[p1] == keys[p1 - 1];
  const bool entered = head && cur < rows;                    // by a run that began before
  bool through = false, leaves = false;                        // that run goes on behind the group; another one does
  float in[V], acc[V];                                         // the sum of that run here; of the current run
#pragma unroll
  for (int i = 0; i < V; i++) in[i] = acc[i] = 0.0f;
  constexpr int U = 8;
  for (int b = p0; b < p1; b += U) {
    unsigned k[U];
    RowPiece<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int p = min(b + u, p1 - 1);
      k[u] = keys[p];
      v[u] = row_load<T, V>(dout + (long)order[p] * dstride, c, k[u] < rows ? D : 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (b + u >= p1) break;
      if (k[u] != cur) {                                       // a run ends inside the group
        if (head) {
#pragma unroll
          for (int i = 0; i < V; i++) in[i] = acc[i];
        } else {
#pragma unroll
          for (int i = 0; i < V; i++) acc[i] *= scale;
          row_store<G, V, true>(grad + (long)cur * D, c, D, acc);
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
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] *= scale;
      row_store<G, V, true>(grad + (long)cur * D, c, D, acc);
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
  float* mine = part + (long)blockIdx.x * 2 * D;
  if (gi == 0 && entered) {                                    // the run that enters the share
    for (int j = 1; j < 4 && on[j - 1]; j++)
#pragma unroll
      for (int i = 0; i < V; i++) in[i] += met[j][wl][i];
    row_store<float, V>(mine, c, D, in);
  }
  if (leaves) {
    for (int j = w + 1; j < 4 && through; j++) {
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] += met[j][lane][i];
      through = on[j];
    }
    if (through) {
      row_store<float, V>(mine + D, c, D, acc);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] *= scale;
      row_store<G, V, true>(grad + (long)cur * D, c, D, acc);
    }
  }
}

// grid (`each` shares each, pieces of the columns): a run that crosses the end of the share in which it begins is finished here.
// Its partial rows are added by sub-groups of lanes, each every (256 >> ls)-th of them, and the sub-groups are joined in order through LDS.
template <typename G, int V>
__global__ __launch_bounds__(256) void embed_join_kernel(const unsigned* __restrict__ keys, int n, unsigned rows, int D, int ls,
                                                         int share, float scale, G* __restrict__ grad, const float* __restrict__ part,
                                                         int each) {
  __shared__ float red[256][V + 1];
  const int tid = threadIdx.x, sub = tid >> ls, subs = 256 >> ls;
  const int c = (int)blockIdx.y * (V << ls) + (tid & ((1 << ls) - 1)) * V;
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
    const int end = emb_lower_bound_wave(keys, p1, n, cur + 1u);
    const int m = (end - 1) / share - g + 1;                   // partial rows: [g][1], [g + 1][0], [g + 2][0], ...
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.0f;
    if (c < D) {
#pragma unroll 8
      for (int i = sub; i < m; i += subs) {
        const RowPiece<float, V> v = row_load<float, V>(part + ((long)(g + i) * 2 + (i == 0 ? 1 : 0)) * D, c, D);
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] += v.e[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; e++) red[tid][e] = acc[e];
    __syncthreads();
    if (sub == 0 && c < D) {
      for (int s = 1; s < min(subs, m); s++)
#pragma unroll
        for (int e = 0; e < V; e++) acc[e] += red[(s << ls) + tid][e];
#pragma unroll
      for (int e = 0; e < V; e++) acc[e] *= scale;
      row_store<G, V, true>(grad + (long)cur * D, c, D, acc);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------------------------
// limits that keep every grid below 2^32 threads (a group of up to 64 lanes per 16 tokens, 4 lanes per table row) and places in 32 bits
#define EMB_MAX_COLS 65536
#define EMB_MAX_TOKENS (1L << 27)
#define EMB_MAX_ROWS (1L << 29)

struct EmbPlan {
  bool ranked;
  int passes, bits, tiles, ls, group, shares;
  size_t keys[2], order[2], hist, total, part, bytes;
};

static EmbPlan emb_plan(long n, long rows, int cols, int vec) {
  EmbPlan p;
  p.ranked = n <= RANK_MAX;
  int need = 1;
  while (need < 32 && ((unsigned long)rows >> need) != 0) need++;         // keys 0 .. rows
  p.passes = p.ranked ? 0 : (need + 9) / 10;
  p.bits = p.ranked ? 0 : (need + p.passes - 1) / p.passes;
  p.tiles = (int)((n + TILE - 1) / TILE);
  p.ls = row_lanes_log2(cols, vec);
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
  for (int i = 0; i < 2; i++) {
    p.keys[i] = take(i == 0 || p.passes > 1 ? 4 * (size_t)n : 0);
    p.order[i] = take(i == 0 || p.passes > 1 ? 4 * (size_t)n : 0);
  }
  p.hist = take(p.ranked ? 0 : (size_t)p.tiles * (4u << p.bits));
  p.total = take(p.ranked ? 0 : 4u << p.bits);
  p.part = take(p.shares > 1 ? (size_t)p.shares * 2 * cols * 4 : 0);
  p.bytes = at;
  return p;
}

static inline bool emb_type(int dtype) { return dtype == NS_F16 || dtype == NS_BF16 || dtype == NS_F32; }

template <typename T, typename I>
static void emb_forward(const void* table, long tstride, const void* ids, void* out, long n, long rows, int cols, float scale,
                        hipStream_t s) {
  const int ls = row_lanes_log2(cols, row_vec<T>());
  hipLaunchKernelGGL((embed_fwd_kernel<T, I>), dim3((unsigned)((n + (256 >> ls) * EMB_U - 1) / ((256 >> ls) * EMB_U))), dim3(256), 0, s,
                     (const T*)table, tstride, (const I*)ids, (T*)out, n, (unsigned)rows, cols, ls, scale);
}

extern "C" int ns_embedding_forward(const void* table, long table_stride, const void* ids, int ids_are_64, void* out, int dtype,
                                    long n, long rows, int cols, float scale, void* stream) {
  NS_REQUIRE(n >= 0 && rows >= 0, "ns_embedding_forward: bad shape");
  NS_REQUIRE(emb_type(dtype), "ns_embedding_forward: dtype %d is not NS_F16, NS_BF16 or NS_F32", dtype);
  if (n == 0) return NS_OK;
  NS_REQUIRE(ids && out && (table || rows == 0), "ns_embedding_forward: null pointer");
  NS_REQUIRE(n <= EMB_MAX_TOKENS && rows <= EMB_MAX_ROWS && cols >= 1 && cols <= EMB_MAX_COLS && table_stride >= 0,
             "ns_embedding_forward: bad shape (n %ld <= 2^27, rows %ld <= 2^29, cols %d in 1 .. %d)", n, rows, cols, EMB_MAX_COLS);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    if (ids_are_64) emb_forward<T, int64_t>(table, table_stride, ids, out, n, rows, cols, scale, s);
    else emb_forward<T, int32_t>(table, table_stride, ids, out, n, rows, cols, scale, s);
  };
  if (dtype == NS_F16) go((_Float16)0);
  else if (dtype == NS_BF16) go((rw_bf16)0.0f);
  else go(0.0f);
  NS_CHECK_LAUNCH("embed_fwd_kernel");
  return NS_OK;
}

extern "C" size_t ns_embedding_backward_workspace_bytes(long n, long rows, int cols, int dtype) {
  if (n <= 0 || n > EMB_MAX_TOKENS || rows < 0 || rows > EMB_MAX_ROWS || cols < 1 || cols > EMB_MAX_COLS) return 0;
  return emb_plan(n, rows, cols, dtype == NS_F32 ? 4 : 8).bytes;
}

template <typename I>
static void emb_sort(const EmbPlan& p, const I* ids, char* ws, int n, unsigned rows, const unsigned** keys, const int** order,
                     hipStream_t s) {
  unsigned* k[2] = {(unsigned*)(ws + p.keys[0]), (unsigned*)(ws + p.keys[1])};
  int* o[2] = {(int*)(ws + p.order[0]), (int*)(ws + p.order[1])};
  if (p.ranked) {
    hipLaunchKernelGGL(embed_rank_kernel<I>, dim3((n + 63) / 64), dim3(64 * RANK_WAVES), 0, s, ids, n, rows, k[0], o[0]);
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
    if (n <= ONE_MAX) {
      hipLaunchKernelGGL(embed_pass_kernel<I>, dim3(p.tiles), dim3(TILE), (2 * ONE_COPIES + ONE_WAVES / 2) * sizeof(int) << p.bits, s, ids, ki, oi, n, rows,
                         i * p.bits, p.bits, k[i & 1], o[i & 1]);
      ki = k[i & 1];
      oi = o[i & 1];
      continue;
    }
    hipLaunchKernelGGL(embed_hist_kernel<I>, dim3(p.tiles), dim3(256), 0, s, ids, ki, (long)n, rows, i * p.bits, bins, hist);
    hipLaunchKernelGGL(embed_prefix_kernel, dim3((bins + 63) / 64), dim3(1024), 0, s, hist, p.tiles, bins, total);
    hipLaunchKernelGGL(embed_scatter_kernel<I>, dim3(p.tiles), dim3(256), 0, s, ids, ki, oi, (long)n, rows, i * p.bits, p.bits, hist,
                       total, k[i & 1], o[i & 1]);
    ki = k[i & 1];
    oi = o[i & 1];
  }
  *keys = ki;
  *order = oi;
}

template <typename T, typename G>
static void emb_sums(const EmbPlan& p, const T* dout, long dstride, const unsigned* keys, const int* order, int n, unsigned rows,
                     int cols, float scale, G* grad, float* part, hipStream_t s) {
  constexpr int V = row_vec<T>();
  const int zero_blocks = (int)(((long)rows + 4 * ZERO_ROWS - 1) / (4 * ZERO_ROWS));
  const int col_blocks = (cols + (V << p.ls) - 1) / (V << p.ls), share = p.group * (256 >> p.ls);
  hipLaunchKernelGGL((embed_sum_kernel<T, G>), dim3(p.shares + zero_blocks, col_blocks), dim3(256), 0, s, dout, dstride, keys, order, n,
                     rows, cols, p.ls, p.group, p.shares, scale, grad, part);
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
  NS_REQUIRE(grad && (n == 0 || (dout && ids && ws)), "ns_embedding_backward: null pointer");
  NS_REQUIRE(n <= EMB_MAX_TOKENS && rows <= EMB_MAX_ROWS && cols >= 1 && cols <= EMB_MAX_COLS && dout_stride >= 0,
             "ns_embedding_backward: bad shape (n %ld <= 2^27, rows %ld <= 2^29, cols %d in 1 .. %d)", n, rows, cols, EMB_MAX_COLS);
  const EmbPlan p = emb_plan(n, rows, cols, dtype == NS_F32 ? 4 : 8);
  NS_REQUIRE(n == 0 || ws_bytes >= p.bytes, "ns_embedding_backward: workspace of %zu bytes, %zu needed", ws_bytes, p.bytes);
  NS_REQUIRE(((uintptr_t)ws % 16) == 0, "ns_embedding_backward: the workspace needs 16-byte alignment");
  hipStream_t s = (hipStream_t)stream;
  const unsigned* keys = nullptr;
  const int* order = nullptr;
  if (n > 0) {
    if (ids_are_64) emb_sort(p, (const int64_t*)ids, (char*)ws, (int)n, (unsigned)rows, &keys, &order, s);
    else emb_sort(p, (const int32_t*)ids, (char*)ws, (int)n, (unsigned)rows, &keys, &order, s);
    NS_CHECK_LAUNCH("embedding_backward: sort");
  }
  auto go = [&](auto t) {
    using T = decltype(t);
    float* part = (float*)((char*)ws + p.part);
    if (grad_dtype == NS_F32)
      emb_sums<T, float>(p, (const T*)dout, dout_stride, keys, order, (int)n, (unsigned)rows, cols, scale, (float*)grad, part, s);
    else
      emb_sums<T, T>(p, (const T*)dout, dout_stride, keys, order, (int)n, (unsigned)rows, cols, scale, (T*)grad, part, s);
  };
  if (dtype == NS_F16) go((_Float16)0);
  else if (dtype == NS_BF16) go((rw_bf16)0.0f);
  else go(0.0f);
  NS_CHECK_LAUNCH("embedding_backward: sums");
  return NS_OK;
}
