// Log probabilities of given classes (or tokens), with the entropy and the best alternatives of every row, and their gradient
// (gfx950).
//
//   m = max_j x_j, S = sum_j exp(x_j - m), T = sum_j (x_j - m) exp(x_j - m)
//   lse = m + log S,  logp = (x_t - m) - log S,  H = -sum_j p_j log p_j = log S - T / S
//   the k largest x_j, equal ones in the order of their index, as (j, (x_j - m) - log S)
//   dx_j = sum over the given ones of g (d_j,idx - p_j)  -  g_H p_j (log p_j + H),   p_j = exp(x_j - lse)
//
// Forward: a block (256 threads) holds a SEGMENT of a row in registers as it lies in memory (16-byte vectors, at most 8 a
// thread: 16384 classes in 16 bits), so the logits are read once for all of it.  A short row is one wave's.  The maximum
// of the segment is known before the first exponential, so there is ONE exponential a class.  Alternatives: the k-th
// largest of a wave's 64 lane maxima is a lower bound of the k-th largest value (bit by bit with ballots: 32 compares);
// the vectors that reach the best wave's bound go into a list of LDS, of those the values that do - some dozens - into a
// second one, and an entry's place is the number of larger ones.  Value and index make one 64-bit key (larger value first, then lower index): all keys differ, so
// the order in which lanes append does not matter.  Segments of one row are joined by a second launch.
#include "rowops.h"

#define LP_MAX_TOP LMH_LOG_PROBS_MAX_TOP
#define LP_SEG_VECS 8
#define LP_JOIN_LDS 4096

typedef unsigned long long u64;

// Order of the values as unsigned integers; -0 counts as +0, NaN as the largest.  0 is no value's key.
__device__ __forceinline__ uint32_t lp_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.f);
  if (f != f) return 0xffffffffu;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float lp_unkey(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ u64 lp_pair(uint32_t key, uint32_t index) { return ((u64)key << 32) | (uint32_t)~index; }

// A lower bound of the k-th largest of the 64 lanes' keys (k <= 64): the largest value that k lanes reach, bit by bit, as far as
// the upper 16 bits (of fp32 values: 7 bits of the mantissa; a looser bound only lengthens the list).
__device__ __forceinline__ uint32_t lp_kth_of_wave(uint32_t key, int k) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(key >= c)) >= k) t = c;
  }
  return t;
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp_max_u32(uint32_t v) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
  return w > v ? w : v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = dpp_max_u32<0xB1>(v);
  v = dpp_max_u32<0x4E>(v);
  v = dpp_max_u32<0x141>(v);
  v = dpp_max_u32<0x140>(v);
  auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = s[0] > s[1] ? s[0] : s[1];
  s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return s[0] > s[1] ? s[0] : s[1];
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
  const uint32_t hi = wave_max_u32((uint32_t)(v >> 32));
  const uint32_t lo = wave_max_u32((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0);
  return ((u64)hi << 32) | lo;
}

struct lp_out {
  float *logp, *entropy, *lse, *top;
  int64_t* index;
};

// What a row's sums say.  S == 0: every class is masked (-inf): log p = -inf everywhere, no entropy.
__device__ __forceinline__ void lp_finish_row(const lp_out& o, int64_t row, float m, float S, float T, bool has_target, float xt) {
  const bool empty = S == 0.f;
  const float log_s = empty ? 0.f : logf(S), m0 = empty ? 0.f : m;
  o.lse[row] = empty ? -INFINITY : m + log_s;
  o.entropy[row] = empty ? 0.f : log_s - T / S;
  if (o.logp) o.logp[row] = has_target ? (xt - m0) - log_s : 0.f;
}

template <typename T, typename I>
__device__ __forceinline__ bool lp_target(const T* x, const I* targets, int64_t row, int V, float* xt) {
  *xt = 0.f;
  if (!targets) return false;
  const int64_t t = (int64_t)targets[row];
  if (t < 0) return false;
  *xt = t < V ? to_f32(x[t]) : NAN;         // a class that does not exist: not a number, never a read outside the row
  return true;
}

template <typename T> __device__ __forceinline__ raw16 load_classes(const T* row, int col, int end) {
  constexpr int VEC = row_type<T>::VEC;
  if (col + VEC <= end) return load16(row + col);
  const uint32_t none = __is_same(T, f32_t) ? 0xff800000u : __is_same(T, f16_t) ? 0xfc00fc00u : 0xff80ff80u;
  raw16 r = {none, none, none, none};
  if (col < end) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (col + e < end) {
        if constexpr (VEC == 4) {
          r[e] = __float_as_uint(row[col + e].v);
        } else {
          const uint32_t b = __builtin_bit_cast(uint16_t, row[col + e]), sh = 16 * (e & 1);
          r[e >> 1] = (r[e >> 1] & ~(0xffffu << sh)) | (b << sh);
        }
      }
  }
  return r;
}

// TPR threads a row or segment (64: one wave, no block-wide step; 256: the block), NV vectors a thread.
// Partial results of a segment: stats[(row * segs + seg) * 3] and, sorted, best[(row * segs + seg) * k].
template <typename T, typename I, int TPR, int NV>
__global__ void __launch_bounds__(256)
k_log_probs(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, int64_t rows, int V, int k, int segs, lp_out out,
            float* __restrict__ stats, u64* __restrict__ best) {
  constexpr int VEC = row_type<T>::VEC, SEG = TPR * NV * VEC, GPB = 256 / TPR, WPG = TPR / 64;
  constexpr int LIST = TPR == 64 ? 128 : 512, VLIST = TPR == 64 ? 64 : 256;
  __shared__ float red[3][4];
  __shared__ uint32_t red_key[4];
  __shared__ u64 list[GPB][LIST];
  __shared__ u64 winner[4];
  __shared__ raw16 vlist[GPB][VLIST];
  __shared__ int vcol[GPB][VLIST], vcount[GPB], count[GPB];
  const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR;
  const int64_t unit = (int64_t)blockIdx.x * GPB + grp;         // (row, segment)
  const int64_t row = unit / segs;
  const int seg = (int)(unit % segs);
  const bool live = row < rows;                                 // (whole waves: TPR >= 64)
  const int first = seg * SEG;
  const T* xr = x + (live ? row : 0) * ldx;
  const int end = live ? V : 0;
  // (behind the end: -inf, which no maximum and no sum sees)
  raw16 r[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) r[v] = load_classes(xr, first + (v * TPR + lane) * VEC, end);
  if (lane == 0) count[grp] = vcount[grp] = 0;

  // ---- maximum, of every vector and of all (fmaxf passes over not-a-number: those rows show in S)
  float vmax[NV], mine = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    vmax[v] = elem<T>(r[v], 0);
#pragma unroll
    for (int e = 1; e < VEC; ++e) vmax[v] = fmaxf(vmax[v], elem<T>(r[v], e));
    mine = fmaxf(mine, vmax[v]);
  }
  float m = reduce64(mine, op_max());
  uint32_t bound = 0;
  if (k > 0) bound = lp_kth_of_wave(lp_key(mine), k);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      red[0][threadIdx.x >> 6] = m;
      red_key[threadIdx.x >> 6] = bound;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      m = fmaxf(m, red[0][w]);
      bound = red_key[w] > bound ? red_key[w] : bound;
    }
  }
  const float m0 = m == -INFINITY ? 0.f : m;

  // ---- sums, and the entries of the list
  float S = 0.f, W = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float z = elem<T>(r[v], e) - m0, p = __expf(z);
      S += p;
      W = fmaf(fmaxf(z, -200.f), p, W);          // (p = 0 below -104: -inf must not meet it)
    }
    if (k > 0 && lp_key(vmax[v]) >= bound) {       // the vector goes to the list whole
      const int at = atomicAdd(&vcount[grp], 1);
      if (at < VLIST) {
        vlist[grp][at] = r[v];
        vcol[grp][at] = first + (v * TPR + lane) * VEC;
      }
    }
  }
  S = reduce64(S, op_add());
  W = reduce64(W, op_add());
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      red[1][threadIdx.x >> 6] = S;
      red[2][threadIdx.x >> 6] = W;
    }
  }
  __syncthreads();
  if constexpr (TPR > 64) {
    S = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    W = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  }
  float log_s = 0.f;
  if (segs == 1) {
    log_s = S == 0.f ? 0.f : logf(S);
    if (live && lane == 0) {
      float xt;
      const bool has = lp_target<T, I>(xr, targets, row, V, &xt);
      lp_finish_row(out, row, m, S, W, has, xt);
    }
  } else if (live && lane == 0) {
    float* st = stats + unit * 3;
    st[0] = m;
    st[1] = S;
    st[2] = W;
  }
  if (k == 0 || !live) return;          // (block-uniform but for waves of TPR = 64, which meet no barrier below)

  auto emit = [&](int rank, u64 pair) {
    if (segs == 1) {
      out.index[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)pair;
      const uint32_t key = (uint32_t)(pair >> 32);
      out.top[row * k + rank] = key == 0xffffffffu ? NAN : (lp_unkey(key) - m0) - log_s;
    } else {
      best[unit * k + rank] = pair;
    }
  };
  const int nv = vcount[grp];
  int n = LIST + 1;
  if (nv <= VLIST) {
    for (int i = lane; i < nv * VEC; i += TPR) {
      const int col = vcol[grp][i / VEC] + i % VEC;
      const uint32_t key = lp_key(to_f32(reinterpret_cast<const T*>(&vlist[grp][0])[i]));
      if (key >= bound && col < end) {
        const int at = atomicAdd(&count[grp], 1);
        if (at < LIST) list[grp][at] = lp_pair(key, (uint32_t)col);
      }
    }
    if constexpr (TPR > 64) __syncthreads();
    n = count[grp];
  }
  if (n <= LIST && S == S) {
    for (int i = lane; i < n; i += TPR) {
      const u64 p = list[grp][i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[grp][j] > p;
      if (rank < k) emit(rank, p);
    }
    if (segs > 1)                       // a last segment shorter than k
      for (int i = n + lane; i < k; i += TPR) emit(i, 0);
    return;
  }
  // many equal values, most large ones in few lanes, or not-a-number among them: k times the largest key below the last one
  u64 last = ~0ull;
  for (int rank = 0; rank < k; ++rank) {
    u64 mx = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int col = first + (v * TPR + lane) * VEC + e;
        if (col < end) {
          const u64 p = lp_pair(lp_key(elem<T>(r[v], e)), (uint32_t)col);
          if (p < last && p > mx) mx = p;
        }
      }
    mx = wave_max_u64(mx);
    if constexpr (TPR > 64) {
      __syncthreads();                  // (the last round's winners are read)
      if ((threadIdx.x & 63) == 0) winner[threadIdx.x >> 6] = mx;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = winner[w] > mx ? winner[w] : mx;
    }
    if (lane == 0) emit(rank, mx);
    last = mx;
  }
}

// One block a row: the segments' lists go to LDS (every list is sorted), then the first wave joins the sums and takes k times
// the largest of the lists' heads.
template <typename T, typename I>
__global__ void __launch_bounds__(256)
k_log_probs_join(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, int64_t rows, int V, int k, int segs, lp_out out,
                 const float* __restrict__ stats, const u64* __restrict__ best) {
  extern __shared__ u64 lists[];        // [segs][k] when that is at most LP_JOIN_LDS entries
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const u64* b = best + row * segs * k;
  const bool in_lds = segs <= 64 && segs * k <= LP_JOIN_LDS;
  if (in_lds) {
    for (int i = threadIdx.x; i < segs * k; i += blockDim.x) lists[i] = b[i];
    if (blockDim.x > 64) __syncthreads();
  }
  if (threadIdx.x >= 64) return;
  const float* st = stats + row * segs * 3;
  float m = -INFINITY;
  for (int s = lane; s < segs; s += 64) m = fmaxf(m, st[3 * s]);
  m = reduce64(m, op_max());
  const float m0 = m == -INFINITY ? 0.f : m;
  float S = 0.f, W = 0.f;
  for (int s = lane; s < segs; s += 64) {
    const float ms = st[3 * s], Ss = st[3 * s + 1], Ws = st[3 * s + 2];
    if (Ss != 0.f) {                    // a segment of -inf alone adds nothing
      const float d = (ms == -INFINITY ? 0.f : ms) - m0, f = expf(d);
      S = fmaf(f, Ss, S);
      W = fmaf(f, fmaf(f > 0.f ? d : 0.f, Ss, Ws), W);
    }
  }
  S = reduce64(S, op_add());
  W = reduce64(W, op_add());
  if (lane == 0) {
    float xt;
    const bool has = lp_target<T, I>(x + row * ldx, targets, row, V, &xt);
    lp_finish_row(out, row, m, S, W, has, xt);
  }
  if (k == 0) return;
  const float log_s = S == 0.f ? 0.f : logf(S);
  auto emit = [&](int rank, u64 pair) {
    const uint32_t key = (uint32_t)(pair >> 32);
    out.index[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)pair;
    out.top[row * k + rank] = key == 0xffffffffu ? NAN : (lp_unkey(key) - m0) - log_s;
  };
  u64 last = ~0ull, mine = 0;           // lane r keeps the alternative of rank r (k <= 64)
  if (in_lds) {
    int pos = 0;
    u64 head = lane < segs ? lists[lane * k] : 0;
    for (int rank = 0; rank < k; ++rank) {
      const u64 mx = wave_max_u64(head);
      if (lane == rank) mine = mx;
      if (head == mx && lane < segs) {
        ++pos;
        head = pos < k ? lists[lane * k + pos] : 0;
      }
    }
  } else {
    for (int rank = 0; rank < k; ++rank) {      // the largest entry below the last one
      u64 mx = 0;
      for (int64_t i = lane; i < (int64_t)segs * k; i += 64) {
        const u64 p = b[i];
        if (p < last && p > mx) mx = p;
      }
      mx = wave_max_u64(mx);
      if (lane == rank) mine = mx;
      last = mx;
    }
  }
  if (lane < k) emit(lane, mine);
}

// Gradient: a thread's vectors of one row, then the given classes' own entries, written whole (p, entropy and every
// gradient given for that class, in the order target, alternative 0, 1, ...) by one thread each, behind a barrier.
template <typename T, typename I>
__global__ void __launch_bounds__(256)
k_log_probs_bwd(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, const float* __restrict__ lse,
                const float* __restrict__ entropy, const float* __restrict__ g_logp, const float* __restrict__ g_entropy,
                const int64_t* __restrict__ index, const float* __restrict__ g_top, int64_t rows, int V, int k, int chunk, int chunks,
                T* __restrict__ dx) {
  constexpr int VEC = row_type<T>::VEC;
  const int64_t row = blockIdx.x / chunks;
  const int first = (int)(blockIdx.x % chunks) * chunk;
  const int end = V - first < chunk ? V : first + chunk;
  const T* xr = x + row * ldx;
  T* dr = dx + row * (int64_t)V;
  const float l = lse[row];
  const bool empty = l == -INFINITY;
  const int64_t t = targets && g_logp ? (int64_t)targets[row] : -1;
  float gt = t >= 0 ? g_logp[row] : 0.f;
  if (t >= V) gt = NAN;
  float G = gt;
  for (int i = 0; i < k; ++i) G += g_top[row * k + i];
  const float h = g_entropy ? entropy[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f;
  auto value = [&](float f) {
    const float lp = f - l, p = __expf(lp);
    return p > 0.f || p != p ? -p * fmaf(gh, lp + h, G) : 0.f;
  };
  for (int col = first + (int)threadIdx.x * VEC; col < end; col += 256 * VEC) {
    const raw16 r = load_cols(xr, col, end);
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = empty ? 0.f : value(elem<T>(r, e));
    store_cols(dr, col, end, o);
  }
  if (empty) return;
  __syncthreads();
  for (int i = (int)threadIdx.x - 1; i < k; i += 256) {
    const int64_t at = i < 0 ? t : index[row * k + i];
    if (at < first || at >= end) continue;
    float g = at == t ? gt : 0.f;
    for (int j = 0; j < k; ++j) g += index[row * k + j] == at ? g_top[row * k + j] : 0.f;
    dr[at] = from_f32<T>(value(to_f32(xr[at])) + g);
  }
}

// ------------------------------------------------------------------------------------------------------- host ----
struct lp_plan { int tpr, nv, segs; };
static lp_plan lp_pick(int64_t rows, int V, int vec) {
  lp_plan p;
  if (V <= 64 * vec * 2) {
    p.tpr = 64;
    p.nv = V <= 64 * vec ? 1 : 2;
    p.segs = 1;
    return p;
  }
  p.tpr = 256;
  p.nv = LP_SEG_VECS;
  while (p.nv > 1 && (256 * vec * (p.nv / 2) >= V || rows * ((V + (int64_t)256 * vec * p.nv - 1) / (256 * vec * p.nv)) < 512)) p.nv /= 2;
  p.segs = (V + (int64_t)256 * vec * p.nv - 1) / (256 * vec * p.nv);
  return p;
}

extern "C" size_t lmh_log_probs_workspace_bytes(int64_t rows, int V, int dtype, int top) {
  if (rows <= 0 || V <= 0 || V > LMH_ROW_MAX_COLS || top < 0 || top > LP_MAX_TOP) return 0;
  const lp_plan p = lp_pick(rows, V, dtype == LMH_F32 ? 4 : 8);
  if (p.segs == 1) return 0;
  return lmh_align_up((size_t)rows * p.segs * 3 * sizeof(float), 256) + lmh_align_up((size_t)rows * p.segs * top * sizeof(u64), 256) + 256;
}

template <typename T, typename I>
static void lp_fwd_launch(const void* x, int64_t ldx, const void* targets, int64_t rows, int V, int k, const lp_out& o, void* ws, hipStream_t st) {
  const lp_plan p = lp_pick(rows, V, row_type<T>::VEC);
  float* stats = (float*)ws;
  u64* best = ws ? (u64*)((char*)ws + lmh_align_up((size_t)rows * p.segs * 3 * sizeof(float), 256)) : nullptr;
  const int64_t units = rows * p.segs;
  const unsigned blocks = (unsigned)(p.tpr == 64 ? (units + 3) / 4 : units);
#define LP_FWD(TPR_, NV_)                                                                                                   \
  lmh_launch((k_log_probs<T, I, TPR_, NV_>), dim3(blocks), dim3(256), 0, st, (const T*)x, ldx, (const I*)targets, rows, V, k, p.segs, o, \
             stats, best)
  if (p.tpr == 64) { if (p.nv == 1) LP_FWD(64, 1); else LP_FWD(64, 2); }
  else if (p.nv == 1) LP_FWD(256, 1);
  else if (p.nv == 2) LP_FWD(256, 2);
  else if (p.nv == 4) LP_FWD(256, 4);
  else LP_FWD(256, 8);
#undef LP_FWD
  if (p.segs > 1)       // few entries: one wave a row
    lmh_launch((k_log_probs_join<T, I>), dim3((unsigned)rows), dim3(p.segs * k > 512 ? 256 : 64),
               (unsigned)(p.segs <= 64 && p.segs * k <= LP_JOIN_LDS ? p.segs * k * sizeof(u64) : 0), st, (const T*)x, ldx, (const I*)targets, rows, V, k, p.segs, o,
               (const float*)stats, (const u64*)best);
}

static int lp_bwd_chunk(int64_t rows, int V, int vec) {
  const int unit = 256 * vec;
  int chunk = 4 * unit;
  while (chunk > unit && rows * ((V + chunk - 1) / chunk) < 1024) chunk /= 2;
  return chunk;
}
static int64_t lp_bwd_chunks(int64_t rows, int V, int vec) {
  const int chunk = lp_bwd_chunk(rows, V, vec);
  return ((int64_t)V + chunk - 1) / chunk;
}

template <typename T, typename I>
static void lp_bwd_launch(const void* x, int64_t ldx, const void* targets, const float* lse, const float* entropy, const float* g_logp,
                          const float* g_entropy, const int64_t* index, const float* g_top, int64_t rows, int V, int k, void* dx,
                          hipStream_t st) {
  const int chunk = lp_bwd_chunk(rows, V, row_type<T>::VEC);
  const int chunks = (int)lp_bwd_chunks(rows, V, row_type<T>::VEC);
  lmh_launch((k_log_probs_bwd<T, I>), dim3((unsigned)(rows * chunks)), dim3(256), 0, st, (const T*)x, ldx, (const I*)targets, lse, entropy,
             g_logp, g_entropy, index, g_top, rows, V, k, chunk, chunks, (T*)dx);
}

#define LP_TYPES(FN, ...)                                                                                                   \
  do {                                                                                                                      \
    if (dtype == LMH_F32) { if (index64) FN<f32_t, int64_t>(__VA_ARGS__); else FN<f32_t, int32_t>(__VA_ARGS__); }           \
    else if (dtype == LMH_F16) { if (index64) FN<f16_t, int64_t>(__VA_ARGS__); else FN<f16_t, int32_t>(__VA_ARGS__); }      \
    else { if (index64) FN<bf16_t, int64_t>(__VA_ARGS__); else FN<bf16_t, int32_t>(__VA_ARGS__); }                          \
  } while (0)

static bool lp_args_ok(int dtype, int64_t rows, int V, int64_t ldx, int top) {
  if (dtype != LMH_F32 && dtype != LMH_F16 && dtype != LMH_BF16) return false;
  if (rows < 0 || V <= 0 || V > LMH_ROW_MAX_COLS || ldx < V || top < 0 || top > LP_MAX_TOP || top > V) return false;
  // a launch has fewer than 2^32 threads
  const int vec = dtype == LMH_F32 ? 4 : 8;
  if (rows > 0x3ffffff) return false;
  const lp_plan p = lp_pick(rows, V, vec);
  return rows * p.segs / (256 / p.tpr) < 0xffffff && rows * lp_bwd_chunks(rows, V, vec) < 0xffffff;
}

extern "C" int lmh_log_probs_fwd(const void* x, int64_t ldx, int dtype, const void* targets, int index64, int64_t rows, int V, int top,
                                 float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_index, void* ws, size_t ws_bytes,
                                 lmh_stream_t stream) {
  LMH_CHECK_ARG(lp_args_ok(dtype, rows, V, ldx, top));
  if (rows == 0) return LMH_OK;
  LMH_CHECK_ARG(x && entropy && lse && (!targets == !logp) && (top == 0 || (top_logp && top_index)));
  const size_t need = lmh_log_probs_workspace_bytes(rows, V, dtype, top);
  if (need && (!ws || ws_bytes < need)) {
    lmh_set_error("lmh_log_probs_fwd: workspace too small");
    return LMH_ERR_WORKSPACE;
  }
  const lp_out o = {logp, entropy, lse, top_logp, top_index};
  hipStream_t st = (hipStream_t)stream;
  LP_TYPES(lp_fwd_launch, x, ldx, targets, rows, V, top, o, ws, st);
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}

extern "C" int lmh_log_probs_bwd(const void* x, int64_t ldx, int dtype, const void* targets, int index64, const float* lse,
                                 const float* entropy, const float* g_logp, const float* g_entropy, const int64_t* top_index,
                                 const float* g_top, int64_t rows, int V, int top, void* dx, lmh_stream_t stream) {
  LMH_CHECK_ARG(lp_args_ok(dtype, rows, V, ldx, top));
  if (rows == 0) return LMH_OK;
  LMH_CHECK_ARG(x && lse && dx && (!g_logp || targets) && (!g_entropy || entropy) && (top == 0 || (top_index && g_top)));
  hipStream_t st = (hipStream_t)stream;
  LP_TYPES(lp_bwd_launch, x, ldx, targets, lse, entropy, g_logp, g_entropy, top_index, g_top, rows, V, top, dx, st);
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}
