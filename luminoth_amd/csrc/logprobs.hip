// Log probabilities of given classes (or tokens), with the entropy and the best alternatives of every row, and their gradient
// (gfx950).
//
//   m = max_j x_j, S = sum_j exp(x_j - m), T = sum_j (x_j - m) exp(x_j - m)
//   lse = m + log S,  logp = (x_t - m) - log S,  H = -sum_j p_j log p_j = log S - T / S
//   the k largest x_j, equal ones in the order of their index, as (j, (x_j - m) - log S)
//   dx_j = sum over the given ones of g (d_j,idx - p_j)  -  g_H p_j (log p_j + H),   p_j = exp(x_j - lse)
//
// Forward: a block (256 threads) takes one row, or a part of it, SEGMENT by segment: 16-byte vectors as they lie in memory, at most
// 4 a thread (8192 classes in 16 bits), read once for all of it.  A short row is one wave's.  Every thread keeps a maximum and
// sums of its own over its segments (rescaled when the maximum grows: one more exponential for 32) and they are joined at the
// end: no barrier inside the loop.
// Alternatives: the k-th largest of a wave's 64 lane maxima so far is a lower bound of the k-th largest value (bit by bit with
// ballots: 16 compares); vectors that reach the bound go into a list of LDS whole - some dozens, fewer and fewer from segment to
// segment -, of those the values that reach the last bound into a second one, and an entry's place there is the number of
// larger ones.  Value and index make one 64-bit key (larger value first, then lower index): all keys differ, so the order in
// which lanes append does not matter.  Parts of one row are joined by a second launch.
// Bound by HBM.  Measured: 2048 x 100003 f16 with 8 alternatives 91-102 us = 4.0-4.5 TB/s, 4096 x 65536 bf16 98-134 us (4.0-5.5 TB/s:
// what still lies in the last-level cache), its gradient 169 us = 6.4 TB/s read and written, 777 x 32003 fp32 with 3 alternatives
// 22 + 4 us and 36 us; 1 x 131072 bf16 with 20 6 + 7 us and 4000 x 81 fp32 with 5 5.6 us, latency.
#include <algorithm>
#include <cmath>

#include "rowops.h"

#define LP_MAX_TOP LMH_LOG_PROBS_MAX_TOP
#define LP_SEG_VECS 4             // 64 registers: eight blocks a compute unit (8: 88 registers, 2-4 % slower)

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

template <typename T> __device__ __forceinline__ raw16 load_classes(const T* row, int col, int end) {       // -inf behind the end
  return load_cols(row, col, end, __is_same(T, f32_t) ? 0xff800000u : __is_same(T, f16_t) ? 0xfc00fc00u : 0xff80ff80u);
}

// TPR threads a row or a part of one (64: one wave, no block-wide step; 256 or 1024: the block), NV vectors a thread and segment, `run`
// segments a part.  Results of a part: stats[(row * parts + part) * 3] and, sorted, best[(row * parts + part) * k].
template <typename T, typename I, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
k_log_probs(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, int64_t rows, int V, int k, int run, int parts, lp_out out,
            float* __restrict__ stats, u64* __restrict__ best) {
  constexpr int VEC = row_type<T>::VEC, SEG = TPR * NV * VEC, GPB = TPR > 256 ? 1 : 256 / TPR, NW = TPR > 256 ? TPR / 64 : 4;
  constexpr int LIST = TPR == 64 ? 128 : 512, VLIST = TPR == 64 ? 128 : TPR == 256 ? 512 : 1024;
  constexpr uint32_t NONE = 0x007fffffu;                        // the key of -inf
  __shared__ float red[3][NW];
  __shared__ uint32_t bounds[NW];
  __shared__ u64 list[GPB][LIST];
  __shared__ u64 winner[NW];
  __shared__ raw16 vlist[GPB][VLIST];
  __shared__ int vcol[GPB][VLIST], vcount[GPB], count[GPB];
  const int lane = threadIdx.x & (TPR - 1), grp = threadIdx.x / TPR, wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * GPB + grp;         // (row, part)
  const int64_t row = parts == 1 ? unit : unit / parts;
  const int first = parts == 1 ? 0 : (int)(unit % parts) * run * SEG;
  const bool live = row < rows;                                 // (whole waves: TPR >= 64)
  const T* xr = x + (live ? row : 0) * ldx;
  const int64_t stop = (int64_t)first + (int64_t)run * SEG;
  const int end = !live ? 0 : stop < V ? (int)stop : V;         // of this part
  if (lane == 0) count[grp] = vcount[grp] = 0;
  if ((threadIdx.x & 63) == 0) bounds[wave] = 0;
  __syncthreads();

  float m = -INFINITY, S = 0.f, W = 0.f;                        // this thread's
  uint32_t top = 0, own = 0;                                    // this lane's largest key, this wave's bound
  for (int base = first; base < end; base += SEG) {
    // (behind the end: -inf, which no maximum and no sum sees)
    raw16 r[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) r[v] = load_classes(xr, base + (v * TPR + lane) * VEC, end);
    // maximum, of every vector and of all (fmaxf passes over not-a-number: those rows show in S)
    float vmax[NV], mine = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vmax[v] = elem<T>(r[v], 0);
#pragma unroll
      for (int e = 1; e < VEC; ++e) vmax[v] = fmaxf(vmax[v], elem<T>(r[v], e));
      mine = fmaxf(mine, vmax[v]);
    }
    // (what was unpacked for the maxima is unpacked again below: kept, it would take a register a class)
#pragma unroll
    for (int v = 0; v < NV; ++v) asm volatile("" : "+v"(r[v]));
    if (mine > m) {                                             // sums of (x - m): exp(d) of them, and d more in each
      const float d = m - mine, f = S > 0.f ? __expf(d) : S;    // (S = 0: nothing there; not-a-number stays)
      W = S > 0.f ? f * fmaf(fmaxf(d, -200.f), S, W) : W;
      S *= f;
      m = mine;
    }
    const float m0 = m == -INFINITY ? 0.f : m;
    // entries of the list: what k values of this wave's earlier segments reach is not needed (those come first), nor what is
    // below k values of this segment and those, or of another wave
    uint32_t low = 0xffffffffu;
    if (k > 0) {
      const uint32_t key = lp_key(mine);
      top = key > top ? key : top;
      if (__any(key > own && key > NONE)) {
        const uint32_t now = lp_kth_of_wave(top, k);
        low = own + 1 > NONE + 1 ? own + 1 : NONE + 1;
        low = now > low ? now : low;
        own = now;
        if constexpr (TPR > 64) {                               // (others' bounds may be old: old ones hold too)
          volatile uint32_t* b = bounds;
          if ((threadIdx.x & 63) == 0) b[wave] = now;
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const uint32_t o = b[w];
            low = o > low ? o : low;
          }
        }
      }
    }
    // (keys and values are in the same order: one compare of values a vector)
    const float low_value = low == 0xffffffffu ? INFINITY : lp_unkey(low);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = elem<T>(r[v], e) - m0, p = __expf(z);
        S += p;
        W = fmaf(fmaxf(z, -200.f), p, W);          // (p = 0 below -104: -inf must not meet it)
      }
      if (vmax[v] >= low_value && low != 0xffffffffu) {
        const int at = atomicAdd(&vcount[grp], 1);
        if (at < VLIST) {
          vlist[grp][at] = r[v];
          vcol[grp][at] = base + (v * TPR + lane) * VEC;
        }
      }
    }
  }

  // ---- the threads' sums joined
  float M = reduce64(m, op_max());
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      red[0][wave] = M;
      bounds[wave] = own;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, red[0][w]);
  }
  const float m0 = M == -INFINITY ? 0.f : M;
  if (S > 0.f) {
    const float d = m - m0, f = __expf(d);
    W = f * fmaf(fmaxf(d, -200.f), S, W);
    S *= f;
  }
  S = reduce64(S, op_add());
  W = reduce64(W, op_add());
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      red[1][wave] = S;
      red[2][wave] = W;
    }
    __syncthreads();
    S = W = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      S += red[1][w];
      W += red[2][w];
    }
  }
  float log_s = 0.f;
  if (parts == 1) {
    log_s = S == 0.f ? 0.f : logf(S);
    if (live && lane == 0) {
      float xt;
      const bool has = lp_target<T, I>(xr, targets, row, V, &xt);
      lp_finish_row(out, row, M, S, W, has, xt);
    }
  } else if (live && lane == 0) {
    float* st = stats + unit * 3;
    st[0] = M;
    st[1] = S;
    st[2] = W;
  }
  if (k == 0 || !live) return;          // (block-uniform but for waves of TPR = 64, which meet no barrier below)

  auto emit = [&](int rank, u64 pair) {
    if (parts == 1) {
      out.index[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)pair;
      const uint32_t key = (uint32_t)(pair >> 32);
      out.top[row * k + rank] = key == 0xffffffffu ? NAN : (lp_unkey(key) - m0) - log_s;
    } else {
      best[unit * k + rank] = pair;
    }
  };
  uint32_t bound = own;
  if constexpr (TPR > 64) {
#pragma unroll
    for (int w = 0; w < NW; ++w) bound = bounds[w] > bound ? bounds[w] : bound;
  }
  bound = bound > NONE ? bound : NONE + 1;
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
  } else if (S == S) {                  // more vectors than the list holds: once more through the part, with the last bound
    for (int col = first + lane * VEC; col < end; col += TPR * VEC) {
      const raw16 r = load_classes(xr, col, end);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t key = lp_key(elem<T>(r, e));
        if (key >= bound && col + e < end) {
          const int at = atomicAdd(&count[grp], 1);
          if (at < LIST) list[grp][at] = lp_pair(key, (uint32_t)(col + e));
        }
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
    // fewer than k classes above -inf: those of -inf in the order of their index, then (a short part) none
    if (n < k && lane < 64) {
      int at = n;
      for (int base = first; base < end && at < k; base += 64) {
        const int col = base + lane;
        const bool none = col < end && lp_key(to_f32(xr[col])) == NONE;
        const u64 mask = __ballot(none);
        const int rank = at + __popcll(mask & ((1ull << lane) - 1));
        if (none && rank < k) emit(rank, lp_pair(NONE, (uint32_t)col));
        at += __popcll(mask);
      }
      if (at + lane < k) emit(at + lane, 0);
    }
    return;
  }
  // many equal values or not-a-number among them: k times the largest key below the last one (the first time: of all - not-a-number
  // at class 0 has the largest there is)
  u64 last = 0;
  for (int rank = 0; rank < k; ++rank) {
    u64 mx = 0;
    for (int col = first + lane * VEC; col < end; col += TPR * VEC) {
      const raw16 r = load_classes(xr, col, end);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const u64 p = lp_pair(lp_key(elem<T>(r, e)), (uint32_t)(col + e));
        if (col + e < end && (rank == 0 || p < last) && p > mx) mx = p;
      }
    }
    mx = wave_max_u64(mx);
    if constexpr (TPR > 64) {
      __syncthreads();                  // (the last round's winners are read)
      if ((threadIdx.x & 63) == 0) winner[wave] = mx;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) mx = winner[w] > mx ? winner[w] : mx;
    }
    if (lane == 0) emit(rank, mx);
    last = mx;
  }
}

// One block a row: the parts' lists go to LDS (every list is sorted), then the first wave joins the sums and takes k times
// the largest of the lists' heads.
template <typename T, typename I>
__global__ void __launch_bounds__(256)
k_log_probs_join(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, int64_t rows, int V, int k, int segs, lp_out out,
                 const float* __restrict__ stats, const u64* __restrict__ best) {
  extern __shared__ u64 lists[];        // [segs][k]: with alternatives a row has at most 64 parts
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const u64* b = best + row * segs * k;
  if (k > 0) {
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
  u64 mine = 0;                         // lane r keeps the alternative of rank r (k <= 64)
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
  if (lane < k) emit(lane, mine);
}

// Gradient: a thread's vectors of one row, then the given classes' own entries, written whole (p, entropy and every
// gradient given for that class, in the order target, alternative 0, 1, ...) by one thread each, behind a barrier.  A short row is
// one wave's, a longer one is cut into `chunks` of one block each.
//
// lse = m + log S has been rounded to fp32: up to |lse| 2^-24 of log S is lost, and every p of the row would be off by that factor (logits
// around 1e4: 5e-4).  Where that is more than 2^-20 (|lse| >= LP_LSE_EXACT) the block sums exp(x - lse) over the whole row, which is what was lost.
// A sum that differs from 1 by more than the rounding belongs to an lse of other classes too (a vocabulary in shards): that counts as given.
// That costs an exponential a class of the row in every block, so there one block takes the chunks of `join`, all of a row's while
// LP_JOINED blocks are left: 4096 x 65536 bf16 with logits around 1000 301 us (187 around 0; every block for itself 710), 777 x 32003 fp32 53
// (32; 141, 79 with 2048 blocks left), 100 x 131072 bf16 51 (11; 58).
#define LP_LSE_EXACT 32.f
#define LP_JOINED 512
template <typename T, typename I, int TPR>
__global__ void __launch_bounds__(256)
k_log_probs_bwd(const T* __restrict__ x, int64_t ldx, const I* __restrict__ targets, const float* __restrict__ lse,
                const float* __restrict__ entropy, const float* __restrict__ g_logp, const float* __restrict__ g_entropy,
                const int64_t* __restrict__ index, const float* __restrict__ g_top, int64_t rows, int V, int k, int chunk, int chunks,
                int join, T* __restrict__ dx) {
  constexpr int VEC = row_type<T>::VEC;
  const int lane = threadIdx.x & (TPR - 1);
  const int64_t row = TPR == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x / chunks;
  if (TPR == 64 && row >= rows) return;                         // (no barrier below)
  int first = TPR == 64 ? 0 : (int)(blockIdx.x % chunks) * chunk;
  int end = V - first < chunk ? V : first + chunk;
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
  float rest = 0.f;                                             // log S = (lse - m) + rest
  if (fabsf(l) >= LP_LSE_EXACT && fabsf(l) < INFINITY) {        // (the same for all threads of a row)
    __shared__ float red[4];
    if (TPR > 64) {
      // (another one from row to row: every eighth block runs on the same die)
      const int c = (int)(blockIdx.x % chunks), c0 = c / join * join, n = min(join, chunks - c0);
      if (c - c0 != (int)(((uint32_t)row * 2654435769u >> 8) % (uint32_t)n)) return;                     // (the whole block)
      first = c0 * chunk;
      end = V - first < (int64_t)chunk * n ? V : first + chunk * n;
    }
    float s = 0.f;
#pragma unroll 4
    for (int col = lane * VEC; col < V; col += TPR * VEC) {
      const raw16 r = load_classes(xr, col, V);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += __expf(elem<T>(r, e) - l);
    }
    s = reduce_row<TPR>(s, op_add(), red);
    const float lost = logf(s);
    if (fabsf(lost) <= fabsf(l) * 0x1p-23f + 0x1p-19f) rest = lost;
  }
  auto value = [&](float f) {
    const float lp = f - l - rest, p = __expf(lp);
    return p > 0.f || p != p ? -p * fmaf(gh, lp + h, G) : 0.f;
  };
  for (int col = first + lane * VEC; col < end; col += TPR * VEC) {
    const raw16 r = load_cols(xr, col, end);
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = empty ? 0.f : value(elem<T>(r, e));
    store_cols(dr, col, end, o);
  }
  if (empty) return;
  // the vectors' stores come first: those of the block, or of this wave
  if constexpr (TPR == 64) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else __syncthreads();
  for (int i = lane - 1; i < k; i += TPR) {
    const int64_t at = i < 0 ? t : index[row * k + i];
    if (at < first || at >= end) continue;
    float g = at == t ? gt : 0.f;
    for (int j = 0; j < k; ++j) g += index[row * k + j] == at ? g_top[row * k + j] : 0.f;
    dr[at] = from_f32<T>(value(to_f32(xr[at])) + g);
  }
}

// ------------------------------------------------------------------------------------------------------- host ----
struct lp_plan { int tpr, nv, run, parts; };
// A short row is one wave's.  A longer one is cut into segments, shorter ones while there are fewer than two blocks for a compute
// unit; of full segments a block takes several behind each other (the list of alternatives then lets fewer and fewer vectors in,
// and there is less to join: 2048 rows of 100003 classes in f16 with 8 alternatives took 162 us segment by segment, 91 us with
// whole rows = 4.5 TB/s).
#define LP_BLOCKS 2048     // blocks the chip holds at a time, eight a compute unit
// Up to 256 rows of at most this many bytes go to one large block each: 1 x 60000 bf16 takes 11 us, as in parts with the launch that
// joins them (5 + 5 us), but one launch of the host's; 40 x 130000 19 us against 7 + 5.
#define LP_ALONE 131072
static lp_plan lp_pick(int64_t rows, int V, int vec, int top) {
  lp_plan p;
  p.run = p.parts = 1;
  if (V <= 64 * vec * 2) {
    p.tpr = 64;
    p.nv = V <= 64 * vec ? 1 : 2;
    return p;
  }
  if (rows <= 256 && (int64_t)V * (16 / vec) <= LP_ALONE) {
    p.tpr = 1024;
    p.nv = LP_SEG_VECS;
    while (p.nv > 1 && 1024 * vec * (p.nv / 2) >= V) p.nv /= 2;
    p.run = (V + 1024 * vec * p.nv - 1) / (1024 * vec * p.nv);
    return p;
  }
  p.tpr = 256;
  p.nv = LP_SEG_VECS;
  auto segments = [&](int nv) { return ((int64_t)V + 256 * vec * nv - 1) / (256 * vec * nv); };
  while (p.nv > 1 && (256 * vec * (p.nv / 2) >= V || (rows * segments(p.nv) < 512 && segments(p.nv / 2) <= 64))) p.nv /= 2;
  const int64_t segs = segments(p.nv);
  p.parts = (int)segs;
  // n segments of random values put at most about 4.8 top (log n + 0.6) vectors into the list of 512: as many as make 400
  const int most = top ? (int)std::min(1e6, std::max(1.0, std::exp(std::min(20.0, 400 / (4.8 * top) - 0.6)))) : 1000000;
  if (p.nv == LP_SEG_VECS) {
    // as many parts as take the least time: rounds of blocks times segments of one, and 0.4 of a segment for what a block costs
    float least = 1e30f;
    for (int64_t parts = (segs + most - 1) / most, lo = parts; parts <= segs && (parts == lo || rows * (parts - 1) < 4 * LP_BLOCKS); ++parts) {
      const float t = (float)((rows * parts + LP_BLOCKS - 1) / LP_BLOCKS) * ((float)((segs + parts - 1) / parts) + 0.4f);
      if (t < least) {
        least = t;
        p.parts = (int)parts;
      }
    }
  }
  if (top > 0 && p.parts > 64) p.parts = 64;      // a lane of the joining wave has one list
  p.run = (int)((segs + p.parts - 1) / p.parts);         // even parts
  return p;
}

extern "C" size_t lmh_log_probs_workspace_bytes(int64_t rows, int V, int dtype, int top) {
  if (rows <= 0 || V <= 0 || V > LMH_ROW_MAX_COLS || top < 0 || top > LP_MAX_TOP) return 0;
  const lp_plan p = lp_pick(rows, V, dtype == LMH_F32 ? 4 : 8, top);
  if (p.parts == 1) return 0;
  return lmh_align_up((size_t)rows * p.parts * 3 * sizeof(float), 256) + lmh_align_up((size_t)rows * p.parts * top * sizeof(u64), 256) + 256;
}

template <typename T, typename I>
static void lp_fwd_launch(const void* x, int64_t ldx, const void* targets, int64_t rows, int V, int k, const lp_out& o, void* ws, hipStream_t st) {
  const lp_plan p = lp_pick(rows, V, row_type<T>::VEC, k);
  float* stats = (float*)ws;
  u64* best = ws ? (u64*)((char*)ws + lmh_align_up((size_t)rows * p.parts * 3 * sizeof(float), 256)) : nullptr;
  const int64_t units = rows * p.parts;
  const unsigned blocks = (unsigned)(p.tpr == 64 ? (units + 3) / 4 : units);      // (256 or 1024 threads a part)
#define LP_FWD(TPR_, NV_)                                                                                                   \
  lmh_launch((k_log_probs<T, I, TPR_, NV_>), dim3(blocks), dim3(TPR_ > 256 ? TPR_ : 256), 0, st, (const T*)x, ldx, (const I*)targets, rows, V, k, p.run, p.parts, \
             o, stats, best)
  if (p.tpr == 64) { if (p.nv == 1) LP_FWD(64, 1); else LP_FWD(64, 2); }
  else if (p.tpr == 1024) { if (p.nv == 1) LP_FWD(1024, 1); else if (p.nv == 2) LP_FWD(1024, 2); else LP_FWD(1024, 4); }
  else if (p.nv == 1) LP_FWD(256, 1);
  else if (p.nv == 2) LP_FWD(256, 2);
  else LP_FWD(256, 4);
#undef LP_FWD
  if (p.parts > 1)       // few entries: one wave a row
    lmh_launch((k_log_probs_join<T, I>), dim3((unsigned)rows), dim3(p.parts * k > 512 ? 256 : 64),
               (unsigned)(p.parts * k * sizeof(u64)), st, (const T*)x, ldx, (const I*)targets, rows, V, k, p.parts, o,
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
  const int join = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, rows * chunks / LP_JOINED));
#define LP_BWD(TPR_, BLOCKS_)                                                                                               \
  lmh_launch((k_log_probs_bwd<T, I, TPR_>), dim3((unsigned)(BLOCKS_)), dim3(256), 0, st, (const T*)x, ldx, (const I*)targets, lse, entropy, \
             g_logp, g_entropy, index, g_top, rows, V, k, chunk, chunks, join, (T*)dx)
  if (V <= 64 * row_type<T>::VEC * 2) LP_BWD(64, (rows + 3) / 4);
  else LP_BWD(256, rows * chunks);
#undef LP_BWD
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
  if (rows >= 0xffffff) return false;
  const lp_plan p = lp_pick(rows, V, vec, top);
  return rows * p.parts / (p.tpr == 64 ? 4 : 1) < 0xffffff && rows * lp_bwd_chunks(rows, V, vec) < 0xffffff;
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
