// Orthogonalised updates by Newton-Schulz products, for a whole list of matrices at a time (gfx950, matrix cores).
//
//   X = U / max(|U|_F, eps), taken wide (m x n, m <= n);   `steps` times:  A = X X',  X <- p(A) X,  p(A) = a I + b A + c A A
//   a = 3.4445, b = -4.7750, c = 2.0315 (the published quintic: every singular value is driven to about 1)
//   optimizer:  g' = gscale g + wd w,  v = mu v + g',  U = g' + mu v (Nesterov) or v,  w -= lr scale X
//
// Arithmetic.  Small singular values grow by a = 3.44 a step, 485 times in five: 16-bit products would return noise in those
// directions, so the products have fp32 accuracy.  Every operand is held as the sum of two f16 values, hi = f16(x) and
// lo = f16(x - hi): 11 + 1 + 11 bits of x, an error of 2^-24 of its binade.  A product takes three matrix instructions (hi lo,
// lo hi, hi hi; lo lo is below 2^-24) with fp32 accumulation: 3 instead of the 6 of a bf16 split, and 2500 / 3 TFLOP/s
// against 157 of the fp32 instructions.  f16's range is enough because everything here is bounded in the spectral norm, which
// bounds the entries: |X| <= 1.25, |A| <= 1.6, |b I + c A| <= 4.8, |p| <= 3.5, products of three p <= 41; fixed powers of two
// put those below 65504, the largest that do.
// What the fixed scale costs: lo ends at 2^-24, so an entry of X is off by up to 2^-40 whatever its size (a power of two less for the
// others), and small rows lose bits that fp32 would keep: of 300 x 1000 with rows graded from 1 to 1e-6, in units of the row's own
// norm, 7e-7 at 1e-4 of the largest, 6e-6 at 1e-5, 6e-5 at 1e-6 (fp32: 3e-7; with scales a quarter as large four times as much); rows
// down to 1e-3 are as exact as in fp32.
//
// Long matrices (n >= 2 m).  The steps are polynomials in A, which commute: A <- p A p and Q <- p Q take m x m products only, and
// X <- Q X comes every second or third step: of 15 m m n multiplications in five steps 6 are left.  A's error grows by up to
// a^2 = 11.9 a step where A is small (there p hardly depends on it: |b| / a of it), so A is taken anew from X after three
// steps at most.  Relative errors after five steps, of random matrices, against float64 (the same in fp32, step by step in X: 0.9e-6 for
// 20 x 41, 1.4 for 100 x 220, 2.2 for 250 x 600, 3.4 for 1000 x 2100): one step at a time 1.0, 0.8, 1.1, 1.5e-6; two 2.1, 1.9, 1.2,
// 1.8; three 2.9, 2.8, 2.3, 1.9.  So a matrix takes three with a short side of 256, two with one of 128, and X by X goes what is smaller
// or not long (there A has little or nothing to save).  That goes by its own sides, whatever else is in the list: three steps for all
// of a list with one large matrix had squares of 16 beside it off by 5.6e-6, 7 times as much as fp32 (now 0.8e-6).  The three kinds
// advance side by side, a launch for all of them, and the five products with X of one meet the others' where they can: the 42
// matrices of a ResNet-50 detector take 28 launches, 488 us (three steps for all of them: 22 and 444; one: 589).  One matrix of few tiles
// takes as long either way (1024 x 320 100 us with three and with one, 200 x 420 82 and 77), eight of them do not (320 x 1024 199 and
// 219).
//
// Layout.  An operand lies in memory as the matrix instruction takes it ("planes"): [32 rows][16 k] units of hi then lo, 64
// lanes x 16 bytes each, k units of one row block after each other.  Tiles go to LDS with lane-linear 16-byte DMA and come
// back with ds_read_b128 at lane * 16: no bank conflicts, no address arithmetic.  A result leaves the accumulators as
// planes again: with its own rows along k straight from the registers (two lane-half swaps), the other way round through
// LDS.  All products are then row . row products.  Rows and columns are padded with zeros to whole tiles.
//
// Everything m x m is symmetric: only tiles on and above the diagonal are computed.  Launches take all matrices of the list.
// Products with too few tiles for the chip (a long k), and the tiles that a last round of blocks would leave over, are split
// along k; their parts are joined, in order, by a launch of their own.
//
// Measured (five steps): 4096 x 4096 fp32 3.9-4.05 ms, products with X 356 us = 1160 TFLOP/s of f16 instructions, symmetric ones 205 us = 1040;
// 1024 x 320 bf16 98-100 us in 19 launches; the 42 matrices of a ResNet-50 detector, a whole optimizer step, 488 us in 28.
#include <algorithm>
#include <tuple>
#include <type_traits>
#include <vector>

#include "rowops.h"

#define MU_A 3.4445f
#define MU_B -4.7750f
#define MU_C 2.0315f
// scales of what is stored as f16 pairs (powers of two)
#define MU_SX 32768.f     // X
#define MU_SG 32768.f     // A, p A
#define MU_SC 8192.f      // b I + c A, eigenvalues in [b, b + 1.6 c]
#define MU_SP 16384.f     // p(A)
#define MU_SQ 1024.f      // products of up to three of them
#define MU_MAX_GROUPS 24  // of one launch (kernel arguments: under 4 KB together)
#define MU_MAX_JOBS 44
// up to this many tiles of 64 x 64: tiles of 32 x 32 with four waves on each (one matrix, all steps: 1024 x 320, 15 tiles, 165 -> 121 us;
// 512 x 1024, 36 tiles, 188 -> 138; 1024 x 2048, 136 tiles, 356 -> 291; no gain from there on: 1408 x 1500, 253 tiles, 448 and 443;
// the 42 matrices of a ResNet-50 detector, 328 tiles, 13.3 us a launch both)
#define MU_SMALL 160
#define MU_SMALL_X 256        // ... of the products with X
// Two tiles of 128 x 128 in one of 256 x 128: a unit of 16 k then takes 12 KB of LDS reads and 6 KB of writes a wave for 24 matrix
// instructions instead of 8 + 4 for 12 - with those LDS has as many cycles of work as the matrix cores - (4096 x 4096: 373 -> 356 us a
// product = 1160 TFLOP/s of f16 instructions).  Where rounds of blocks cost more than that gains, or k is short and the rest of a
// block's work counts (42 matrices of m = 128 to 512: 50 -> 53 us), 128 x 128 stays.
#define MU_NORM_BLOCKS 512
#define MU_NORM_ELEMS 2048    // at least this many per block of k_mu_norm

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The matrices of one shape in one launch.  Places in the workspace and sizes of buffers are counted in units of 256 bytes; a
// matrix's buffers are given from its start (-1: none).
struct mu_task {
  uint32_t off, stride;
  int32_t m, n, pm, pn, tall;
  int32_t count, first;            // matrices, the first one's place in the table of pointers
  int32_t l, r, d0, d1, norm, aux;
  int32_t whole, splits;           // tiles (of all its matrices) before `whole` are not split along k
  uint32_t slab;                   // partial tiles of the others
  float s0, g0, s1, g1;            // what is stored: accumulator * s + (on the diagonal) g
};
// blk0: the tasks' first blocks, behind each other: the arguments lie in host memory, where a search that goes from task to task
// waits for every one of them (10 us of a 14 us launch).  One task alone has a table of its own, without a search
// (0.8 us a launch: 1024 x 320 114 -> 100 us, 100 x 400 89 -> 73).
template <int N> struct mu_table_of {
  int32_t blk0[N];                 // (unused: the largest integer)
  int32_t tasks;
  mu_task t[N];
};
struct mu_ptrs { const void* g; float* v; void* out; const float* factor; float wd, scale; };      // out: the weights, or the result
template <int N> struct mu_jobs_of { mu_ptrs p[N]; };
typedef mu_table_of<MU_MAX_GROUPS> mu_table;
typedef mu_jobs_of<MU_MAX_JOBS> mu_jobs;

template <int N> __device__ __forceinline__ int mu_find(const mu_table_of<N>& t, int blk) {
  if (N == 1) return 0;
  int i = -1;
#pragma unroll
  for (int k = 0; k < N; ++k) i += blk >= t.blk0[k];
  return i;
}
__device__ __forceinline__ char* mu_at(char* ws, const mu_task& t, int job, int buffer) {
  return ws + ((int64_t)t.off + (int64_t)job * t.stride + buffer) * 256;
}

__device__ __forceinline__ void mu_split(float x, uint16_t* hi, uint16_t* lo) {
  const _Float16 h = (_Float16)x;
  *hi = __builtin_bit_cast(uint16_t, h);
  *lo = __builtin_bit_cast(uint16_t, (_Float16)(x - (float)h));
}

// ---- momentum and the partial sums of the squares ----------------------------------------------------------
// aux: blocks per matrix; d0: the matrix that is orthogonalised, row-major fp32 (the optimizer's; the plain call reads its input)
template <typename T, bool OPT, int N>
__global__ void __launch_bounds__(256)
k_mu_norm(mu_table_of<N> tab, mu_jobs_of<(N == 1 ? 1 : MU_MAX_JOBS)> jobs, char* ws, float mu, int nesterov, float gscale) {
  __shared__ double red[4];
  const int ti = mu_find(tab, blockIdx.x);
  const mu_task& t = tab.t[ti];
  const int local = N == 1 ? blockIdx.x : blockIdx.x - tab.blk0[ti], job = N == 1 ? 0 : local / t.aux, b = N == 1 ? local : local % t.aux;
  const mu_ptrs& p = jobs.p[N == 1 ? 0 : t.first + job];
  const int64_t n = (int64_t)t.m * t.n, stride = (int64_t)t.aux * 256;
  double acc = 0.0;
  if (OPT) {
    float* u = (float*)mu_at(ws, t, job, t.d0);
    const float* g = (const float*)p.g;
    const float* w = (const float*)p.out;
    const float f = p.factor ? *p.factor : 1.f, wd = p.wd;
    auto one = [&](float gi, float wi, float* vi) {
      const float gp = (gi * gscale + wd * wi) * f;
      *vi = mu * *vi + gp;
      const float x = nesterov ? gp + mu * *vi : *vi;
      acc += (double)x * (double)x;
      return x;
    };
    if ((((uintptr_t)g | (uintptr_t)w | (uintptr_t)p.v) & 15) == 0) {
      const int64_t n4 = n >> 2;
      for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n4; i += stride) {
        const float4 gi = reinterpret_cast<const float4*>(g)[i], wi = reinterpret_cast<const float4*>(w)[i];
        float4 vi = reinterpret_cast<const float4*>(p.v)[i], x;
        x.x = one(gi.x, wi.x, &vi.x);
        x.y = one(gi.y, wi.y, &vi.y);
        x.z = one(gi.z, wi.z, &vi.z);
        x.w = one(gi.w, wi.w, &vi.w);
        reinterpret_cast<float4*>(p.v)[i] = vi;
        reinterpret_cast<float4*>(u)[i] = x;
      }
      if (b == 0 && threadIdx.x < (n & 3)) {
        const int64_t i = 4 * n4 + threadIdx.x;
        float v = p.v[i];
        u[i] = one(g[i], w[i], &v);
        p.v[i] = v;
      }
    } else {
      for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n; i += stride) {
        float v = p.v[i];
        u[i] = one(g[i], w[i], &v);
        p.v[i] = v;
      }
    }
  } else {
    constexpr int VEC = row_type<T>::VEC;
    const T* g = (const T*)p.g;
    for (int64_t i = ((int64_t)b * 256 + threadIdx.x) * VEC; i < n; i += 4 * stride * VEC) {
      raw16 r[4];                          // (four loads on their way)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t at = i + u * stride * VEC;
        r[u] = raw16{0, 0, 0, 0};
        if (at < n) r[u] = load_cols(g + at, 0, (int)(n - at < VEC ? n - at : VEC));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc += (double)elem<T>(r[u], e) * (double)elem<T>(r[u], e);
    }
  }
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) ((double*)mu_at(ws, t, job, t.norm))[b] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- X and X' as planes --------------------------------------------------------------------------------------
// One block: 64 x 64 of the matrix as it is stored (rows x cols), padding included.  l: fp32 input (OPT), d0: X, d1: X'
template <typename T, bool OPT, int N>
__global__ void __launch_bounds__(256)
k_mu_planes(mu_table_of<N> tab, mu_jobs_of<(N == 1 ? 1 : MU_MAX_JOBS)> jobs, char* ws, float eps) {
  __shared__ float tile[64][65];
  __shared__ double total;
  const int gi = mu_find(tab, blockIdx.x);
  const mu_task& g = tab.t[gi];
  const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n, prow = g.tall ? g.pn : g.pm, pcol = g.tall ? g.pm : g.pn;
  const int per = (prow / 64) * (pcol / 64), local = N == 1 ? blockIdx.x : blockIdx.x - tab.blk0[gi], job = N == 1 ? 0 : local / per, t = local - job * per;
  const int r0 = (t / (pcol / 64)) * 64, c0 = (t % (pcol / 64)) * 64;
  const void* src = OPT ? (const void*)mu_at(ws, g, job, g.l) : jobs.p[N == 1 ? 0 : g.first + job].g;
  typedef typename std::conditional<OPT, f32_t, T>::type S;
  S raw[16];                               // (sixteen loads on their way; behind the matrix: its last row and column, not used)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = min(r0 + i * 4 + (int)(threadIdx.x >> 6), rows - 1), c = min(c0 + (int)(threadIdx.x & 63), cols - 1);
    raw[i] = ((const S*)src)[(int64_t)r * cols + c];
  }
  if (threadIdx.x < 64) {                  // the matrix's partial sums, in a fixed order
    const double* part = (const double*)mu_at(ws, g, job, g.norm);
    double ss = 0.0;
    for (int i = threadIdx.x; i < g.aux; i += 64) ss += part[i];
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    if (threadIdx.x == 0) total = ss;
  }
  __syncthreads();
  double norm = sqrt(total);
  if (norm < (double)eps) norm = (double)eps;            // (not a number stays one)
  const double inv = (double)MU_SX / norm;               // (may lie outside fp32's range, X does not)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = i * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
    tile[r][c] = r0 + r < rows && c0 + c < cols ? (float)((double)to_f32(raw[i]) * inv) : 0.f;
  }
  __syncthreads();
  // stored rows as rows (k = stored columns): X for a wide matrix, X' for a tall one; and the other way round
  char* by_row = mu_at(ws, g, job, g.tall ? g.d1 : g.d0);
  char* by_col = mu_at(ws, g, job, g.tall ? g.d0 : g.d1);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int unit = wave * 4 + i;           // 0..7: by row, 8..15: by column; (32-row block, 16-k unit) of the tile
    const int rb = (unit >> 2) & 1, kb = unit & 3;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int a = rb * 32 + l31, k = kb * 16 + h * 8 + e;
      uint16_t p, q;
      mu_split(unit < 8 ? tile[a][k] : tile[k][a], &p, &q);
      if (e & 1) { hi[e >> 1] |= (uint32_t)p << 16; lo[e >> 1] |= (uint32_t)q << 16; }
      else { hi[e >> 1] = p; lo[e >> 1] = q; }
    }
    char* out;
    if (unit < 8) out = by_row + ((int64_t)(r0 / 32 + rb) * (pcol / 16) + c0 / 16 + kb) * 2048;
    else out = by_col + ((int64_t)(c0 / 32 + rb) * (prow / 16) + r0 / 16 + kb) * 2048;
    *reinterpret_cast<raw16*>(out + lane * 16) = raw16{hi[0], hi[1], hi[2], hi[3]};
    *reinterpret_cast<raw16*>(out + 1024 + lane * 16) = raw16{lo[0], lo[1], lo[2], lo[3]};
  }
}

// ---- products ------------------------------------------------------------------------------------------------
// The 32 x 32 accumulator (lane: column lane & 31, register i: row (i & 3) + 8 (i >> 2) + 4 (lane >> 5)) as planes:
//  cols: rows = its COLUMNS, k = its rows, two 16-k units at `cols` (+ 2048): pairs of registers are pairs along k, and the lane
//        halves trade so that a lane has eight successive ones;
//  rows: the other way round, if wanted: hi and lo of a value as one word through `turn`, 32 x MU_PITCH words of this wave's LDS.
#define MU_PITCH 40      // writes of the two lane halves (four rows apart) hit the two halves of the banks; 16-byte rows
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void mu_store(const float* v, char* cols, char* rows, int lane, uint32_t* turn) {
  uint32_t hi[8], lo[8];                     // of registers 2 j, 2 j + 1
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const f32x2 x = {v[2 * j], v[2 * j + 1]};
    const f16x2 h = __builtin_convertvector(x, f16x2);
    const f16x2 l = __builtin_convertvector(x - __builtin_convertvector(h, f32x2), f16x2);
    hi[j] = __builtin_bit_cast(uint32_t, h);
    lo[j] = __builtin_bit_cast(uint32_t, l);
  }
  const int l31 = lane & 31, h = lane >> 5;
  if (rows) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = (2 * j & 3) + 8 * (j >> 1) + 4 * h;
      turn[r * MU_PITCH + l31] = __builtin_amdgcn_perm(lo[j], hi[j], 0x05040100);
      turn[(r + 1) * MU_PITCH + l31] = __builtin_amdgcn_perm(lo[j], hi[j], 0x07060302);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    auto a = __builtin_amdgcn_permlane32_swap(hi[4 * u], hi[4 * u + 2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(hi[4 * u + 1], hi[4 * u + 3], false, false);
    auto c = __builtin_amdgcn_permlane32_swap(lo[4 * u], lo[4 * u + 2], false, false);
    auto d = __builtin_amdgcn_permlane32_swap(lo[4 * u + 1], lo[4 * u + 3], false, false);
    *reinterpret_cast<raw16*>(cols + u * 2048 + lane * 16) = raw16{a[0], b[0], a[1], b[1]};
    *reinterpret_cast<raw16*>(cols + u * 2048 + 1024 + lane * 16) = raw16{c[0], d[0], c[1], d[1]};
  }
  if (rows) {
    __builtin_amdgcn_wave_barrier();         // (one wave's LDS accesses are in order)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const raw16* p = reinterpret_cast<const raw16*>(turn + l31 * MU_PITCH + u * 16 + h * 8);
      const raw16 x = p[0], y = p[1];
      *reinterpret_cast<raw16*>(rows + u * 2048 + lane * 16) =
          raw16{__builtin_amdgcn_perm(x[1], x[0], 0x05040100), __builtin_amdgcn_perm(x[3], x[2], 0x05040100),
                __builtin_amdgcn_perm(y[1], y[0], 0x05040100), __builtin_amdgcn_perm(y[3], y[2], 0x05040100)};
      *reinterpret_cast<raw16*>(rows + u * 2048 + 1024 + lane * 16) =
          raw16{__builtin_amdgcn_perm(x[1], x[0], 0x07060302), __builtin_amdgcn_perm(x[3], x[2], 0x07060302),
                __builtin_amdgcn_perm(y[1], y[0], 0x07060302), __builtin_amdgcn_perm(y[3], y[2], 0x07060302)};
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Tile t of the upper triangle of tm x tm tiles: in strips of eight rows, a strip column by column, so that neighbours share
// operands.
__device__ __forceinline__ void mu_triangle(int t, int tm, int* ti, int* tj) {
  int top = 0, high = min(8, tm), all;
  while (t >= (all = high * (high + 1) / 2 + high * (tm - top - high))) {
    t -= all;
    top += high;
    high = min(8, tm - top);
  }
  const int corner = high * (high + 1) / 2;  // the strip's first columns are cut off by the diagonal
  if (t < corner) {
    int c = 0;
    while (t > c) t -= ++c;
    *ti = top + t;
    *tj = top + c;
  } else {
    t -= corner;
    *ti = top + t % high;
    *tj = top + high + t / high;
  }
}

// The accumulator of 32-blocks (rb, cb) of a symmetric result, scaled into its one or two buffers (`only`: one of them), and mirrored
// unless its tile of SQ x SQ blocks lies on the diagonal (all of it is computed).
template <int SQ>
__device__ __forceinline__ void mu_store_symmetric(const mu_task& g, char* ws, int job, const float* acc, int rb, int cb, int lane,
                                                   uint32_t* turn, int only = -1) {
  const int l31 = lane & 31, h = lane >> 5, units = g.pm / 16;
  const bool mirror = rb / SQ != cb / SQ;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = k ? g.d1 : g.d0;
    if (d < 0 || (only >= 0 && k != only)) continue;
    const float s = k ? g.s1 : g.s0, on = k ? g.g1 : g.g0;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = acc[i] * s + (rb == cb && (i & 3) + 8 * (i >> 2) + 4 * h == l31 ? on : 0.f);
    char* out = mu_at(ws, g, job, d);
    mu_store(v, out + ((int64_t)cb * units + rb * 2) * 2048, mirror ? out + ((int64_t)rb * units + cb * 2) * 2048 : nullptr, lane, turn);
  }
}

enum { MU_SYM = 0, MU_APPLY = 1, MU_LAST = 2 };

// One tile of 64 TA x 64 TB of C = L . R' (rows of L and R along k), 4 waves of 32 TA x 32 TB; a ring of DEPTH stages of 16 KU k in LDS.
//  MU_SYM: m x m, tiles of the upper triangle; kinds of operands by r: k runs over aux 16-units.
//  MU_APPLY: l = X' (n x m), r = a polynomial (m x m) -> d0 = X (rows m), d1 = X' (rows n).
//  MU_LAST: the same product into the result (a wide matrix the other way round: lanes then run along stored rows).
template <typename T, int TA, int TB, int KU, int DEPTH, int MODE, bool OPT>
__device__ __forceinline__ void mu_gemm_tile(const mu_table& tab, const mu_jobs* jobs, char* ws, float lr) {
  constexpr int RBA = 2 * TA, RBB = 2 * TB, SU = KU * 2048, STAGE = (RBA + RBB) * SU, NL = (TA + TB) * KU;     // bytes of a stage, a wave's loads
  __shared__ __attribute__((aligned(16))) char smem[DEPTH * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave >> 1, wc = wave & 1, l31 = lane & 31, h = lane >> 5;
  // every eighth block runs on the same die: of 64 blocks, those of a die take eight tiles behind each other, which share operands
  // in its L2
  int blk = blockIdx.x;
  if (blk < (int)(gridDim.x & ~63u)) blk = (blk & ~63) + (blk & 7) * 8 + ((blk >> 3) & 7);
  const int gi = mu_find(tab, blk);
  const mu_task& g = tab.t[gi];
  int u = blk - tab.blk0[gi], split = 0, ti, tj, job;
  const bool turned = MODE == MU_LAST && !g.tall;
  const int rows32 = MODE == MU_SYM || turned ? g.pm / 32 : g.pn / 32, cols32 = turned ? g.pn / 32 : g.pm / 32;      // of the result
  const int tm = (rows32 + RBA - 1) / RBA, tn = cols32 / RBB, per = MODE == MU_SYM ? tm * (tm + 1) / 2 : tm * tn;
  int t;
  if (MODE == MU_SYM && g.whole == 0) {      // all tiles split: a matrix's tiles of one part of k are neighbours
    const unsigned both = (unsigned)per * g.splits, in = (unsigned)u % both;
    job = (unsigned)u / both;
    split = in / (unsigned)per;
    t = in - split * per;
    u = job * per + t;
  } else {
    if (MODE == MU_SYM && u >= g.whole) {
      const unsigned rest = u - g.whole;
      u = g.whole + rest / (unsigned)g.splits;
      split = rest % (unsigned)g.splits;
    }
    job = (unsigned)u / (unsigned)per;
    t = u - job * per;
  }
  if (MODE == MU_SYM) {
    mu_triangle(t, tm, &ti, &tj);
  } else {
    // among the tiles along n and those along m: in strips of eight of the former, a strip one by one of the latter; few of those:
    // the other way round
    const int ta = turned ? tn : tm, tb = turned ? tm : tn;
    const int step = tb > 8 ? 8 : 1, strip = t / (step * tb), in = t - strip * step * tb, high = min(step, ta - strip * step);
    const int row = strip * step + in % high, col = in / high;
    ti = turned ? col : row;
    tj = turned ? row : col;
  }
  const char* L = mu_at(ws, g, job, turned ? g.r : g.l);
  const char* R = mu_at(ws, g, job, turned ? g.l : g.r);
  const int kunits = g.aux;
  int k0 = 0, stages = kunits / KU;
  const bool part = MODE == MU_SYM && u >= g.whole;
  if (part) {                                // splits share the stages evenly
    const unsigned all = stages, parts = g.splits;       // (at most 2^13 stages in 64 parts)
    k0 = (int)(all * split / parts);
    stages = (int)(all * (split + 1) / parts) - k0;
  }
  f32x16 acc[TA][TB];
#pragma unroll
  for (int a = 0; a < TA; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

  typedef __attribute__((address_space(3))) void* lds_ptr;
  typedef const __attribute__((address_space(1))) void* glb_ptr;
  // a stage: RBA row blocks of the left operand and RBB of the right one x KU units x 2 KB; wave w brings in KBs w, w + 4, ...  (Rows
  // behind the last: that one again; their products are dropped.)
  const char* src[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int piece = i * 4 + wave, rb = piece / (2 * KU);
    const int64_t row = rb < RBA ? min(ti * RBA + rb, rows32 - 1) : tj * RBB + rb - RBA;
    src[i] = (rb < RBA ? L : R) + row * kunits * 2048 + (int64_t)k0 * SU + piece % (2 * KU) * 1024 + lane * 16;
  }
  auto issue = [&](int s, int b) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      __builtin_amdgcn_global_load_lds((glb_ptr)(src[i] + (int64_t)s * SU), (lds_ptr)(smem + b * STAGE + (i * 4 + wave) * 1024), 16, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < DEPTH - 1; ++s)
    if (s < stages) issue(s, s);
  int cur = 0;
  for (int s = 0; s < stages; ++s) {
    // this wave's pieces of stage s have landed (DEPTH - 2 later stages may still be on their way); behind the barrier
    // everybody's have, and everybody is done with the stage whose place the next issue takes
    if (DEPTH > 2 && stages - 1 - s >= DEPTH - 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 2) * NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + DEPTH - 1 < stages) issue(s + DEPTH - 1, cur == 0 ? DEPTH - 1 : cur - 1);
    const char* Ls = smem + cur * STAGE + wr * TA * SU + lane * 16;
    const char* Rs = smem + cur * STAGE + RBA * SU + wc * TB * SU + lane * 16;
#pragma unroll
    for (int k = 0; k < KU; ++k) {
      f16x8 lh[TA], ll[TA], rh[TB], rl[TB];
#pragma unroll
      for (int a = 0; a < TA; ++a) lh[a] = *reinterpret_cast<const f16x8*>(Ls + a * SU + k * 2048);
#pragma unroll
      for (int b = 0; b < TB; ++b) rl[b] = *reinterpret_cast<const f16x8*>(Rs + b * SU + k * 2048 + 1024);
#pragma unroll
      for (int a = 0; a < TA; ++a) ll[a] = *reinterpret_cast<const f16x8*>(Ls + a * SU + k * 2048 + 1024);
#pragma unroll
      for (int b = 0; b < TB; ++b) rh[b] = *reinterpret_cast<const f16x8*>(Rs + b * SU + k * 2048);
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[a], rl[b], acc[a][b], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll[a], rh[b], acc[a][b], 0, 0, 0);
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[a], rh[b], acc[a][b], 0, 0, 0);
    }
    cur = cur + 1 == DEPTH ? 0 : cur + 1;
  }

  if constexpr (MODE == MU_SYM) {
    if (part) {
      float* s = (float*)(ws + (int64_t)g.slab * 256) + ((int64_t)(u - g.whole) * g.splits + split) * (RBA * RBB * 1024);
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(s + ((wave * TA + a) * TB + b) * 1024 + q * 256 + lane * 4) =
                make_float4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
      return;
    }
  }
  if constexpr (MODE == MU_LAST) {
    const mu_ptrs& p = jobs->p[g.first + job];
    float* out = (float*)p.out;
    const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n;
    const float scale = OPT ? lr * p.scale * g.s0 : g.s0;
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        const int c = (tj * RBB + wc * TB + b) * 32 + l31, r0 = (ti * RBA + wr * TA + a) * 32 + 4 * h;
        if constexpr (OPT) {                 // sixteen loads on their way, then the stores
          float w[16];
          int64_t at[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = r0 + (i & 3) + 8 * (i >> 2);
            at[i] = r < rows && c < cols ? (int64_t)r * cols + c : 0;
            w[i] = out[at[i]];
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (r0 + (i & 3) + 8 * (i >> 2) < rows && c < cols) out[at[i]] = w[i] - scale * acc[a][b][i];
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = r0 + (i & 3) + 8 * (i >> 2);
            if (r < rows && c < cols) ((T*)p.out)[(int64_t)r * cols + c] = from_f32<T>(scale * acc[a][b][i]);
          }
        }
      }
    return;
  }
  __syncthreads();                           // the stages' LDS is free
  uint32_t* turn = (uint32_t*)smem + wave * 32 * MU_PITCH;
#pragma unroll
  for (int a = 0; a < TA; ++a)
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const int rb = ti * RBA + wr * TA + a, cb = tj * RBB + wc * TB + b;    // 32-blocks of the result
      if (rb >= rows32) continue;
      float v[16];
      if constexpr (MODE == MU_APPLY) {      // rows of the result: n, columns: m
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[a][b][i] * g.s0;
        mu_store(v, mu_at(ws, g, job, g.d0) + ((int64_t)cb * (g.pn / 16) + rb * 2) * 2048,
                 mu_at(ws, g, job, g.d1) + ((int64_t)rb * (g.pm / 16) + cb * 2) * 2048, lane, turn);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[a][b][i];
        mu_store_symmetric<RBB>(g, ws, job, v, rb, cb, lane, turn);
      }
    }
}

template <int TA, int TB, int KU, int DEPTH, int MODE>
__global__ void __launch_bounds__(256, 2)
k_mu_gemm(mu_table tab, char* ws) {
  mu_gemm_tile<f32_t, TA, TB, KU, DEPTH, MODE, false>(tab, nullptr, ws, 0.f);
}
template <typename T, int TA, int TB, int KU, int DEPTH, bool OPT>
__global__ void __launch_bounds__(256, 2)
k_mu_last(mu_table tab, mu_jobs jobs, char* ws, float lr) {
  mu_gemm_tile<T, TA, TB, KU, DEPTH, MU_LAST, OPT>(tab, &jobs, ws, lr);
}

// Few tiles: one of 32 x 32 by four waves, a quarter of k each.  What bounds such a launch is how fast a compute unit gets its operands
// from beyond its die's L2 (some 40 GB/s: another die wrote them; a stage of 32 k of a 64 x 64 tile took 0.42 us, whether two or
// seven more were on their way), so more units with less each: operands come straight to registers (eight units of 16 k on
// their way in a wave), without LDS and barriers, and the quarters are added in LDS, in order.
template <typename T, int MODE, bool OPT, int N, typename J>
__device__ __forceinline__ void mu_small_tile(const mu_table_of<N>& tab, const J* jobs, char* ws, float lr) {
  constexpr int CHUNK = 4;
  __shared__ __attribute__((aligned(16))) float quarter[4][1024];
  __shared__ __attribute__((aligned(16))) uint32_t turns[2][32 * MU_PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
  int blk = blockIdx.x;
  constexpr int RUN = 32;                    // neighbours on a die, as above (8: 4-5 % slower)
  if (blk < (int)(gridDim.x / (8 * RUN) * (8 * RUN))) blk = blk / (8 * RUN) * (8 * RUN) + (blk & 7) * RUN + (blk >> 3) % RUN;
  const int gi = mu_find(tab, blk);
  const mu_task& g = tab.t[gi];
  int u = N == 1 ? blk : blk - tab.blk0[gi], split = 0, ti, tj;
  const int tm = g.pm / 32, tn = g.pn / 32, per = MODE == MU_SYM ? tm * (tm + 1) / 2 : tm * tn;
  const bool part = MODE == MU_SYM && g.whole == 0;
  int job, t;
  if (part) {
    const unsigned both = (unsigned)per * g.splits, in = (unsigned)u % both;
    job = (unsigned)u / both;
    split = in / (unsigned)per;
    t = in - split * per;
    u = job * per + t;
  } else {
    job = (unsigned)u / (unsigned)per;
    t = u - job * per;
  }
  const bool turned = MODE == MU_LAST && !g.tall;
  if (MODE == MU_SYM) {
    mu_triangle(t, tm, &ti, &tj);
  } else {
    const int row = t / tm, col = t % tm;
    ti = turned ? col : row;
    tj = turned ? row : col;
  }
  const int kunits = g.aux;
  int k0 = 0, k1 = kunits;
  if (part) {
    k0 = (int)((unsigned)kunits * split / (unsigned)g.splits);
    k1 = (int)((unsigned)kunits * (split + 1) / (unsigned)g.splits);
  }
  const int u0 = k0 + (k1 - k0) * wave / 4, u1 = k0 + (k1 - k0) * (wave + 1) / 4;
  const char* L = mu_at(ws, g, job, turned ? g.r : g.l) + (int64_t)ti * kunits * 2048 + lane * 16;
  const char* R = mu_at(ws, g, job, turned ? g.l : g.r) + (int64_t)tj * kunits * 2048 + lane * 16;
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  f16x8 f[2][CHUNK][4];
  auto fetch = [&](int at, f16x8 (&d)[CHUNK][4]) {
#pragma unroll
    for (int c = 0; c < CHUNK; ++c) {
      const int64_t off = (int64_t)max(min(at + c, u1 - 1), u0) * 2048;          // (behind the end: the last unit, not used)
      d[c][0] = *reinterpret_cast<const f16x8*>(L + off);
      d[c][1] = *reinterpret_cast<const f16x8*>(L + off + 1024);
      d[c][2] = *reinterpret_cast<const f16x8*>(R + off);
      d[c][3] = *reinterpret_cast<const f16x8*>(R + off + 1024);
    }
  };
  auto work = [&](int at, const f16x8 (&d)[CHUNK][4]) {
#pragma unroll
    for (int c = 0; c < CHUNK; ++c)
      if (at + c < u1) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(d[c][0], d[c][3], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(d[c][1], d[c][2], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(d[c][0], d[c][2], acc, 0, 0, 0);
      }
  };
  if (u0 < u1) {
    fetch(u0, f[0]);
    for (int at = u0; at < u1; at += 2 * CHUNK) {
      if (at + CHUNK < u1) fetch(at + CHUNK, f[1]);
      work(at, f[0]);
      if (at + 2 * CHUNK < u1) fetch(at + 2 * CHUNK, f[0]);
      if (at + CHUNK < u1) work(at + CHUNK, f[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4*>(&quarter[wave][i * 256 + lane * 4]) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
  __syncthreads();
  if (MODE != MU_LAST && wave >= 2) return;
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float4 a = *reinterpret_cast<const float4*>(&quarter[0][i * 256 + lane * 4]);
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 b = *reinterpret_cast<const float4*>(&quarter[w][i * 256 + lane * 4]);
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    v[4 * i] = a.x;
    v[4 * i + 1] = a.y;
    v[4 * i + 2] = a.z;
    v[4 * i + 3] = a.w;
  }
  uint32_t* turn = turns[wave & 1];
  if constexpr (MODE == MU_SYM) {
    if (part) {
      if (wave) return;
      float* s = (float*)(ws + (int64_t)g.slab * 256) + ((int64_t)u * g.splits + split) * 1024;
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(s + q * 256 + lane * 4) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      return;
    }
    mu_store_symmetric<1>(g, ws, job, v, ti, tj, lane, turn, wave);
  } else if constexpr (MODE == MU_APPLY) {
    if (wave) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= g.s0;
    mu_store(v, mu_at(ws, g, job, g.d0) + ((int64_t)tj * (g.pn / 16) + ti * 2) * 2048, mu_at(ws, g, job, g.d1) + ((int64_t)ti * (g.pm / 16) + tj * 2) * 2048,
             lane, turn);
  } else {
    const mu_ptrs& p = jobs->p[g.first + job];
    float* out = (float*)p.out;
    const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n;
    const float scale = OPT ? lr * p.scale * g.s0 : g.s0;
    const int c = tj * 32 + l31, r0 = ti * 32 + 4 * h;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if ((i >> 2) != wave) continue;                  // four rows of every eight a wave
      const int r = r0 + (i & 3) + 8 * (i >> 2);
      if (r < rows && c < cols) {
        if constexpr (OPT) out[(int64_t)r * cols + c] -= scale * v[i];
        else ((T*)p.out)[(int64_t)r * cols + c] = from_f32<T>(scale * v[i]);
      }
    }
  }
}
template <int MODE, int N>
__global__ void __launch_bounds__(256)
k_mu_small(mu_table_of<N> tab, char* ws) {
  mu_small_tile<f32_t, MODE, false>(tab, (const mu_jobs*)nullptr, ws, 0.f);
}
template <typename T, bool OPT, int N>
__global__ void __launch_bounds__(256)
k_mu_small_last(mu_table_of<N> tab, mu_jobs_of<(N == 1 ? 1 : MU_MAX_JOBS)> jobs, char* ws, float lr) {
  mu_small_tile<T, MU_LAST, OPT>(tab, &jobs, ws, lr);
}

// Joins the parts of split tiles (WAVES: four with TW x TW 32-blocks each, or one), one 32 x 32 block of a tile each wave (blk0 counts
// tiles).
template <int TW, int WAVES>
__global__ void __launch_bounds__(64)
k_mu_join(mu_table tab, char* ws) {
  constexpr int W = WAVES == 4 ? 2 : 1, RB = W * TW, SUB = RB * RB;
  __shared__ __attribute__((aligned(16))) uint32_t turn[32 * MU_PITCH];
  const int lane = threadIdx.x, tile = blockIdx.x / SUB, sub = blockIdx.x % SUB;
  const int gi = mu_find(tab, tile);
  const mu_task& g = tab.t[gi];
  const int q0 = tile - tab.blk0[gi], u = g.whole + q0;
  const int tm = g.pm / 32 / RB, per = tm * (tm + 1) / 2, job = u / per;
  int ti, tj;
  mu_triangle(u - job * per, tm, &ti, &tj);
  const float* s = (const float*)(ws + (int64_t)g.slab * 256) + (int64_t)q0 * g.splits * (SUB * 1024) + sub * 1024 + lane * 4;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int k = 0; k < g.splits; ++k, s += SUB * 1024)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(s + q * 256);
      v[4 * q] += f.x;
      v[4 * q + 1] += f.y;
      v[4 * q + 2] += f.z;
      v[4 * q + 3] += f.w;
    }
  const int wave = sub / (TW * TW), a = sub / TW % TW, b = sub % TW;
  mu_store_symmetric<RB>(g, ws, job, v, ti * RB + wave / W * TW + a, tj * RB + wave % W * TW + b, lane, turn);
}

// ------------------------------------------------------------------------------------------------------- host ----
#define MU_SLOTS 512      // blocks of 128 x 128 or 256 x 128 tiles (64 and 72 KB of LDS) the chip holds at a time

static int64_t mu_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct mu_group {
  int m, n, pm, pn, count, first, tall;
  int segment;                         // steps in A behind each other, at most (1: X by X)
  int64_t off, stride;                 // units of 256 bytes
  int x, xt[2], a, c, p, z, q[2], norm, norm_blocks;
};
struct mu_plan {
  std::vector<int> order;              // the caller's jobs, sorted by shape
  std::vector<mu_group> groups;
  int tw;                              // tiles of the products with X: 64 tw
  int64_t slab, slab_units, units;
};

// Splits along k of the symmetric products of a launch: `stages` of 32 k, `tiles` in all.
struct mu_cut { int64_t whole; int splits; };
// Too few tiles: each in as many parts as fill the chip, four stages a part at least.  Else whole, but for what a last round
// would leave over, if that is less than half a round (of 4096 x 4096: 16 of 528 tiles, 1.1 rounds instead of 2).
static mu_cut mu_cut_of(int64_t tiles, int stages, int64_t all_stages, int64_t all_tiles, bool alone, int least) {
  mu_cut c = {tiles, 1};
  if (all_tiles < MU_SLOTS) {
    const int64_t part = std::max<int64_t>(least, (all_stages + MU_SLOTS - 1) / MU_SLOTS);
    c.splits = (int)std::min<int64_t>(64, std::max<int64_t>(1, (stages + part / 2) / part));
    if (c.splits > 1) c.whole = 0;
  } else if (alone) {
    const int64_t rest = tiles % MU_SLOTS;
    const int splits = rest ? (int)std::min<int64_t>(std::min<int64_t>(MU_SLOTS / rest, stages / 4), 16) : 1;
    if (splits > 1) {
      c.whole = tiles - rest;
      c.splits = splits;
    }
  }
  return c;
}

// Tiles (of 128 x 128 and 64 x 64) of the symmetric products of a launch (X X' and those of m x m matrices) or of its products with X,
// and what sides (of 32) its tiles have.
struct mu_counts {
  int64_t grams = 0, squares = 0, xtiles = 0, xtall = 0, xdepth = 0, stages = 0, tiles64 = 0, xtiles64 = 0;
  void add_symmetric(int64_t pm, int64_t count, int64_t units, bool gram) {
    const int64_t t = count * (pm / 128) * (pm / 128 + 1) / 2;
    (gram ? grams : squares) += t;
    if (gram) stages += t * (units / 2);
    tiles64 += count * (pm / 64) * (pm / 64 + 1) / 2;
  }
  void add_apply(int64_t pm, int64_t pn, int64_t count) {
    xtiles += count * (pm / 128) * (pn / 128);
    xdepth += count * (pm / 128) * (pn / 128) * pm;
    xtall += count * (pm / 128) * ((pn / 128 + 1) / 2);
    xtiles64 += count * (pm / 64) * (pn / 64);
  }
  // 64 x 64 while tiles of 128 x 128 would leave places free
  int symmetric() const { return tiles64 <= MU_SMALL ? 1 : squares >= 256 || stages >= 4096 ? 4 : 2; }
  int apply() const {
    if (xtiles64 <= MU_SMALL_X) return 1;
    if (xtiles < 128) return 2;
    const int64_t rounds = (xtiles + MU_SLOTS - 1) / MU_SLOTS, tall = (xtall + MU_SLOTS - 1) / MU_SLOTS;
    return 188 * tall < 100 * rounds && xdepth >= 1024 * xtiles ? 8 : 4;
  }
};

// By a matrix's own sides, whatever else is in the list: its error does not depend on its companions.
static int mu_segment(int m, int n) { return n < 2 * m ? 1 : m >= 256 ? 3 : m >= 128 ? 2 : 1; }

static void mu_make_plan(const lmh_muon_job* jobs, int count, mu_plan* pl) {
  pl->order.resize(count);
  for (int i = 0; i < count; ++i) pl->order[i] = i;
  // by shape, those of the longest products first: a launch's last blocks are short ones
  auto key = [&](int i) {
    const int r = jobs[i].rows, c = jobs[i].cols;
    return std::make_tuple(std::min(r, c), std::max(r, c), r);
  };
  std::stable_sort(pl->order.begin(), pl->order.end(), [&](int a, int b) { return key(a) > key(b); });
  // rows and columns are padded to 128 where a tile of 128 x 128 may be taken (mu_counts), to 64 where none is
  mu_counts gram, square;
  pl->tw = 1;
  for (int i = 0; i < count; ++i) {
    const int m = std::min(jobs[i].rows, jobs[i].cols), n = std::max(jobs[i].rows, jobs[i].cols);
    if (m > 64) pl->tw = 2;
    gram.add_symmetric(mu_up(m, 128), 1, mu_up(n, 128) / 16, true);
    square.add_symmetric(mu_up(m, 128), 1, mu_up(m, 128) / 16, false);
    square.add_apply(mu_up(m, 128), mu_up(n, 128), 1);
  }
  if (gram.symmetric() < 4 && square.symmetric() < 4 && square.apply() < 4) pl->tw = 1;
  const int bt = 64 * pl->tw;
  int64_t off = 0;
  pl->groups.clear();
  for (int s = 0; s < count;) {
    int e = s;
    while (e < count && key(pl->order[e]) == key(pl->order[s])) ++e;
    const lmh_muon_job& j = jobs[pl->order[s]];
    mu_group g;
    g.tall = j.rows > j.cols;
    g.m = g.tall ? j.cols : j.rows;
    g.n = g.tall ? j.rows : j.cols;
    g.pm = (int)mu_up(g.m, bt);
    g.pn = (int)mu_up(g.n, bt);
    g.count = e - s;
    g.first = s;
    g.segment = mu_segment(g.m, g.n);
    const int mn = (int)((int64_t)g.pm * g.pn / 64), mm = (int)((int64_t)g.pm * g.pm / 64);      // 4 bytes a value, units of 256
    int at = 0;
    auto take = [&](int n) { const int r = at; at += n; return r; };
    g.x = take(mn);
    g.xt[0] = take(mn);
    g.xt[1] = take(mn);
    g.a = take(mm);
    g.c = take(mm);
    g.p = take(mm);
    g.z = g.segment > 1 ? take(mm) : -1;
    g.q[0] = g.segment > 1 ? take(mm) : -1;
    g.q[1] = g.segment > 1 ? take(mm) : -1;
    g.norm_blocks = (int)std::min<int64_t>(MU_NORM_BLOCKS, ((int64_t)g.m * g.n + MU_NORM_ELEMS - 1) / MU_NORM_ELEMS);
    g.norm = take((int)((g.norm_blocks * sizeof(double) + 255) / 256));
    g.stride = at;
    g.off = off;
    off += g.stride * g.count;
    pl->groups.push_back(g);
    s = e;
  }
  // a launch's partial tiles: fewer than two for each place on the chip, or 64 parts of the rest of a round
  pl->slab = off;
  pl->slab_units = (int64_t)(2 * MU_SLOTS + 64) * bt * bt * 4 / 256;
  pl->units = off + pl->slab_units;
}

static bool mu_jobs_ok(const lmh_muon_job* jobs, int count) {
  if (!jobs || count <= 0 || count > LMH_MUON_MAX_JOBS) return false;
  for (int i = 0; i < count; ++i)
    if (jobs[i].rows <= 0 || jobs[i].cols <= 0 || jobs[i].rows > LMH_MUON_MAX_DIM || jobs[i].cols > LMH_MUON_MAX_DIM ||
        (int64_t)jobs[i].rows * jobs[i].cols > (1 << 30))
      return false;
  return true;
}

extern "C" size_t lmh_muon_workspace_bytes(const lmh_muon_job* jobs, int count) {
  if (!mu_jobs_ok(jobs, count)) return 0;
  try {
    mu_plan pl;
    mu_make_plan(jobs, count, &pl);
    return pl.units > 0x7fffffff ? 0 : (size_t)pl.units * 256;
  } catch (...) {
    return 0;
  }
}

// Tiles of one product with X: `side` 32-blocks each way; 8: eight along the result's rows and four along its columns.  (The last product's
// rows are those of the matrix as it is stored.)
static int mu_x_tiles(const mu_group& g, int side, bool last) {
  if (side < 8) return g.pm / (32 * side) * (g.pn / (32 * side));
  const int rows = last && !g.tall ? g.pm : g.pn, cols = last && !g.tall ? g.pn : g.pm;
  return (rows + 255) / 256 * (cols / 128);
}

// A launch of one task, or of one matrix: its table and job alone.
static bool mu_alone(const mu_table& t) { return t.tasks == 1 && t.t[0].count == 1; }
static mu_table_of<1> mu_single(const mu_table& t) { return {{0}, 1, {t.t[0]}}; }

class mu_runner {
 public:
  mu_runner(const mu_plan& pl, char* ws, hipStream_t st) : pl_(pl), ws_(ws), st_(st) { memset(&tab_, 0, sizeof(tab_)); }

  // Tasks of the next launch; `fill` sets the operands of one group's task and returns its blocks.
  template <typename F>
  int tasks(const std::vector<const mu_group*>& gs, size_t g0, size_t g1, F fill) {
    int total = 0;
    clear(&tab_);
    for (size_t i = g0; i < g1; ++i) {
      const mu_group& g = *gs[i];
      mu_task& t = tab_.t[tab_.tasks];
      base(g, &t);
      tab_.blk0[tab_.tasks++] = total;
      total += fill(g, &t);
    }
    return total;
  }
  void base(const mu_group& g, mu_task* t) const {
    memset(t, 0, sizeof(*t));
    t->off = (uint32_t)g.off;
    t->stride = (uint32_t)g.stride;
    t->m = g.m;
    t->n = g.n;
    t->pm = g.pm;
    t->pn = g.pn;
    t->tall = g.tall;
    t->count = g.count;
    t->norm = g.norm;
    t->l = t->r = t->d0 = t->d1 = -1;
    t->splits = 1;
    t->whole = 0x7fffffff;
  }

  static void clear(mu_table* t) {
    t->tasks = 0;
    for (int i = 0; i < MU_MAX_GROUPS; ++i) t->blk0[i] = 0x7fffffff;
  }

  struct product { int l, r, d0, d1, units; float s0, g0, s1, g1; bool gram; };
  // Symmetric products of the groups, in tiles of at most 32 `most`.
  void symmetric(const std::vector<std::pair<const mu_group*, product>>& all, int most) {
    mu_counts counts;
    for (size_t i = 0; i < all.size(); ++i) {
      const mu_group& g = *all[i].first;          // (two products of one group count once: 1024 x 2048 274 us, 287 in the larger tiles)
      if (!i || all[i - 1].first != &g) counts.add_symmetric(g.pm, g.count, all[i].second.units, all[i].second.gram);
    }
    const int side = std::min(most, counts.symmetric()), bt = 32 * side;
    for (size_t lo = 0; lo < all.size(); lo += MU_MAX_GROUPS) {
      const size_t hi = std::min(all.size(), lo + MU_MAX_GROUPS);
      int64_t tiles = 0, stages = 0;
      for (size_t i = lo; i < hi; ++i) {
        const int64_t tm = all[i].first->pm / bt, n = tm * (tm + 1) / 2 * all[i].first->count;
        tiles += n;
        stages += n * (all[i].second.units / 2);
      }
      int blocks = 0, joins = 0;
      mu_table join;
      memset(&join, 0, sizeof(join));
      clear(&join);
      clear(&tab_);
      int64_t slab = pl_.slab;
      for (size_t i = lo; i < hi; ++i) {
        const mu_group& g = *all[i].first;
        const product& p = all[i].second;
        mu_task& t = tab_.t[tab_.tasks];
        base(g, &t);
        t.l = p.l;
        t.r = p.r;
        t.d0 = p.d0;
        t.d1 = p.d1;
        t.s0 = p.s0;
        t.g0 = p.g0;
        t.s1 = p.s1;
        t.g1 = p.g1;
        t.aux = p.units;
        const int64_t tm = g.pm / bt, n = tm * (tm + 1) / 2 * g.count;
        mu_cut c = mu_cut_of(n, p.units / 2, stages, tiles, side > 1 && hi - lo == 1, side == 1 ? 32 : side == 2 ? 16 : 8);
        const int64_t need = (n - c.whole) * c.splits * bt * bt * 4 / 256;
        if (slab + need > pl_.slab + pl_.slab_units) c = {n, 1};
        t.whole = (int)c.whole;
        t.splits = c.splits;
        tab_.blk0[tab_.tasks++] = blocks;
        blocks += (int)(c.whole + (n - c.whole) * c.splits);
        if (c.whole < n) {
          t.slab = (uint32_t)slab;
          slab += need;
          join.t[join.tasks] = t;
          join.blk0[join.tasks++] = joins;
          joins += (int)(n - c.whole);
        }
      }
      if (side == 1 && tab_.tasks == 1) lmh_launch((k_mu_small<MU_SYM, 1>), dim3(blocks), dim3(256), 0, st_, mu_single(tab_), ws_);
      else if (side == 1) lmh_launch((k_mu_small<MU_SYM, MU_MAX_GROUPS>), dim3(blocks), dim3(256), 0, st_, tab_, ws_);
      else if (side == 2) lmh_launch((k_mu_gemm<1, 1, 2, 4, MU_SYM>), dim3(blocks), dim3(256), 0, st_, tab_, ws_);
      else lmh_launch((k_mu_gemm<2, 2, 2, 2, MU_SYM>), dim3(blocks), dim3(256), 0, st_, tab_, ws_);
      if (joins) {
        if (side == 1) lmh_launch((k_mu_join<1, 1>), dim3(joins), dim3(64), 0, st_, join, ws_);
        else if (side == 2) lmh_launch((k_mu_join<1, 4>), dim3(joins * 4), dim3(64), 0, st_, join, ws_);
        else lmh_launch((k_mu_join<2, 4>), dim3(joins * 16), dim3(64), 0, st_, join, ws_);
      }
    }
  }
  static int apply_side(const std::vector<const mu_group*>& gs, int most) {
    mu_counts counts;
    for (const mu_group* g : gs) counts.add_apply(g->pm, g->pn, g->count);
    return std::min(most, counts.apply());
  }
  // X <- polynomial X
  template <typename F>
  void apply(const std::vector<const mu_group*>& gs, int most, F operands) {
    const int side = apply_side(gs, most);
    for (size_t lo = 0; lo < gs.size(); lo += MU_MAX_GROUPS) {
      const int nb = tasks(gs, lo, std::min(gs.size(), lo + MU_MAX_GROUPS), [&](const mu_group& g, mu_task* t) {
        operands(g, t);
        t->aux = g.pm / 16;
        return mu_x_tiles(g, side, false) * g.count;
      });
      if (side == 1 && tab_.tasks == 1) lmh_launch((k_mu_small<MU_APPLY, 1>), dim3(nb), dim3(256), 0, st_, mu_single(tab_), ws_);
      else if (side == 1) lmh_launch((k_mu_small<MU_APPLY, MU_MAX_GROUPS>), dim3(nb), dim3(256), 0, st_, tab_, ws_);
      else if (side == 2) lmh_launch((k_mu_gemm<1, 1, 2, 4, MU_APPLY>), dim3(nb), dim3(256), 0, st_, tab_, ws_);
      else if (side == 8) lmh_launch((k_mu_gemm<4, 2, 1, 3, MU_APPLY>), dim3(nb), dim3(256), 0, st_, tab_, ws_);
      else lmh_launch((k_mu_gemm<2, 2, 2, 2, MU_APPLY>), dim3(nb), dim3(256), 0, st_, tab_, ws_);
    }
  }
  // Launches that take the caller's pointers: at most MU_MAX_JOBS matrices of MU_MAX_GROUPS shapes each.
  template <typename F, typename L>
  void with_jobs(const lmh_muon_job* jobs, const std::vector<const mu_group*>& gs, F fill, L launch) {
    size_t i = 0;
    int done = 0;                      // matrices of group i
    while (i < gs.size()) {
      mu_jobs pj;
      memset(&pj, 0, sizeof(pj));
      int n = 0, total = 0;
      clear(&tab_);
      while (i < gs.size() && tab_.tasks < MU_MAX_GROUPS && n < MU_MAX_JOBS) {
        const mu_group& g = *gs[i];
        const int k = std::min(g.count - done, MU_MAX_JOBS - n);
        mu_task& t = tab_.t[tab_.tasks];
        base(g, &t);
        t.off = (uint32_t)(g.off + done * g.stride);
        t.count = k;
        t.first = n;
        tab_.blk0[tab_.tasks++] = total;
        total += fill(g, &t) * k;
        for (int q = 0; q < k; ++q, ++n) {
          const lmh_muon_job& j = jobs[pl_.order[g.first + done + q]];
          pj.p[n] = {j.g, j.v, j.w ? (void*)j.w : j.out, j.factor, j.wd, j.scale};
        }
        done += k;
        if (done == g.count) {
          ++i;
          done = 0;
        }
      }
      launch(dim3(total), tab_, pj);
    }
  }

 private:
  const mu_plan& pl_;
  char* ws_;
  hipStream_t st_;
  mu_table tab_;
};

// The launches of `steps` steps, `segment` of them at most in A behind each other.  flip: which X' is the present one; q: which Q.
enum { MU_GRAM, MU_POLY, MU_MOVE, MU_NEXT, MU_X };
struct mu_launch { int what, k, len, q, flip; };
static std::vector<mu_launch> mu_launches(int steps, int segment) {
  std::vector<mu_launch> l;
  l.reserve(5 * steps);
  for (int done = 0, flip = 0; done < steps; flip = 1 - flip) {
    const int left = steps - done, len = left == 4 ? std::min(2, segment) : std::min(left, segment);
    int q = 0;                         // of a run of several steps: their product so far in q[q]
    l.push_back({MU_GRAM, 0, len, q, flip});
    for (int k = 0; k < len; ++k) {
      l.push_back({MU_POLY, k, len, q, flip});
      if (len == 1) break;
      l.push_back({MU_MOVE, k, len, q, flip});
      if (k > 0) q = 1 - q;
      if (k + 1 < len) l.push_back({MU_NEXT, k, len, q, flip});
    }
    l.push_back({MU_X, 0, len, q, flip});
    done += len;
  }
  return l;
}

template <typename T, bool OPT>
static void mu_run(const lmh_muon_job* jobs, const mu_plan& pl, int steps, float eps, float gscale, float mu, int nesterov, float lr,
                   char* ws, hipStream_t st) {
  mu_runner run(pl, ws, st);
  std::vector<const mu_group*> all;
  bool present[4] = {false, false, false, false};
  for (const mu_group& g : pl.groups) {
    all.push_back(&g);
    present[g.segment] = true;
  }
  run.with_jobs(jobs, all, [](const mu_group& g, mu_task* t) {
    t->aux = g.norm_blocks;
    t->d0 = g.xt[1];                   // (free until the first product with X has been taken)
    return g.norm_blocks;
  }, [&](dim3 nb, const mu_table& tab, const mu_jobs& pj) {
    if (mu_alone(tab)) lmh_launch((k_mu_norm<T, OPT, 1>), nb, dim3(256), 0, st, mu_single(tab), mu_jobs_of<1>{{pj.p[0]}}, ws, mu, nesterov, gscale);
    else lmh_launch((k_mu_norm<T, OPT, MU_MAX_GROUPS>), nb, dim3(256), 0, st, tab, pj, ws, mu, nesterov, gscale);
  });
  run.with_jobs(jobs, all, [](const mu_group& g, mu_task* t) {
    t->aux = g.norm_blocks;
    t->l = g.xt[1];
    t->d0 = g.x;
    t->d1 = g.xt[0];
    return (g.pm / 64) * (g.pn / 64);
  }, [&](dim3 nb, const mu_table& tab, const mu_jobs& pj) {
    if (mu_alone(tab)) lmh_launch((k_mu_planes<T, OPT, 1>), nb, dim3(256), 0, st, mu_single(tab), mu_jobs_of<1>{{pj.p[0]}}, ws, eps);
    else lmh_launch((k_mu_planes<T, OPT, MU_MAX_GROUPS>), nb, dim3(256), 0, st, tab, pj, ws, eps);
  });
  // Matrices of different segments go side by side, a launch of each in every round.  A product with X waits one round where the next
  // but one launch of others is one too: they share it.
  std::vector<mu_launch> seq[4];
  size_t at[4] = {0, 0, 0, 0};
  for (int s = 1; s < 4; ++s)
    if (present[s]) seq[s] = mu_launches(steps, s);
  const int most = pl.tw == 2 ? 8 : 2;
  const float sgg = 1.f / (MU_SX * MU_SX), scg = 1.f / (MU_SC * MU_SG), sgp = 1.f / (MU_SG * MU_SP);
  std::vector<std::pair<const mu_group*, mu_runner::product>> products;
  std::vector<const mu_group*> apply, last;
  products.reserve(2 * all.size());
  for (;;) {
    bool now[4] = {false, false, false, false}, left = false;
    for (int s = 1; s < 4; ++s) {
      if (at[s] >= seq[s].size()) continue;
      left = now[s] = true;
      if (seq[s][at[s]].what != MU_X) continue;
      for (int o = 1; o < 4; ++o)
        if (at[o] + 1 < seq[o].size() && seq[o][at[o]].what != MU_X && seq[o][at[o] + 1].what == MU_X) now[s] = false;
    }
    if (!left) break;
    products.clear();
    apply.clear();
    last.clear();
    for (const mu_group* gp : all) {
      const mu_group& g = *gp;
      if (!now[g.segment]) continue;
      const mu_launch& l = seq[g.segment][at[g.segment]];
      const int units = g.pm / 16;
      switch (l.what) {
        case MU_GRAM:      // A = X X' and b I + c A
          products.push_back({gp, {g.x, g.x, g.a, g.c, g.pn / 16, MU_SG * sgg, 0.f, MU_C * MU_SC * sgg, MU_B * MU_SC, true}});
          break;
        case MU_POLY:      // p = (b I + c A) A + a I; the first of several is their product too
          products.push_back({gp, {g.c, g.a, g.p, l.k == 0 && l.len > 1 ? g.q[0] : -1, units, MU_SP * scg, MU_A * MU_SP, MU_SQ * scg,
                                   MU_A * MU_SQ, false}});
          break;
        case MU_MOVE:      // z = p A unless this is the last of them, Q <- p Q unless it is the first
          if (l.k + 1 < l.len) products.push_back({gp, {g.p, g.a, g.z, -1, units, MU_SG / (MU_SP * MU_SG), 0.f, 0.f, 0.f, false}});
          if (l.k > 0) products.push_back({gp, {g.p, g.q[l.q], g.q[1 - l.q], -1, units, MU_SQ / (MU_SP * MU_SQ), 0.f, 0.f, 0.f, false}});
          break;
        case MU_NEXT:      // A <- z p
          products.push_back({gp, {g.z, g.p, g.a, g.c, units, MU_SG * sgp, 0.f, MU_C * MU_SC * sgp, MU_B * MU_SC, false}});
          break;
        case MU_X:
          (at[g.segment] + 1 == seq[g.segment].size() ? last : apply).push_back(gp);
      }
    }
    if (!products.empty()) run.symmetric(products, most);
    auto operands = [&](const mu_group& g, mu_task* t) {
      const mu_launch& l = seq[g.segment][at[g.segment]];
      t->l = g.xt[l.flip];
      t->r = l.len > 1 ? g.q[l.q] : g.p;
      t->d0 = g.x;
      t->d1 = g.xt[1 - l.flip];
      t->s0 = l.len > 1 ? 1.f / MU_SQ : 1.f / MU_SP;
    };
    if (!apply.empty()) run.apply(apply, most, operands);
    if (!last.empty()) {
      const int side = mu_runner::apply_side(last, most);
      run.with_jobs(jobs, last, [&](const mu_group& g, mu_task* t) {
        operands(g, t);
        t->s0 /= MU_SX;
        t->aux = g.pm / 16;
        return mu_x_tiles(g, side, true);
      }, [&](dim3 nb, const mu_table& tab, const mu_jobs& pj) {
        if (side == 1 && mu_alone(tab))
          lmh_launch((k_mu_small_last<T, OPT, 1>), nb, dim3(256), 0, st, mu_single(tab), mu_jobs_of<1>{{pj.p[0]}}, ws, lr);
        else if (side == 1) lmh_launch((k_mu_small_last<T, OPT, MU_MAX_GROUPS>), nb, dim3(256), 0, st, tab, pj, ws, lr);
        else if (side == 2) lmh_launch((k_mu_last<T, 1, 1, 2, 4, OPT>), nb, dim3(256), 0, st, tab, pj, ws, lr);
        else if (side == 8) lmh_launch((k_mu_last<T, 4, 2, 1, 3, OPT>), nb, dim3(256), 0, st, tab, pj, ws, lr);
        else lmh_launch((k_mu_last<T, 2, 2, 2, 2, OPT>), nb, dim3(256), 0, st, tab, pj, ws, lr);
      });
    }
    for (int s = 1; s < 4; ++s) at[s] += now[s];
  }
}

static int mu_check(const lmh_muon_job* jobs, int count, int steps, float eps, void* ws, size_t ws_bytes, mu_plan* pl) {
  LMH_CHECK_ARG(mu_jobs_ok(jobs, count) && steps >= 1 && steps <= LMH_MUON_MAX_STEPS && eps > 0.f);
  try {
    mu_make_plan(jobs, count, pl);
  } catch (...) {
    lmh_set_error("lmh_muon: out of host memory");
    return LMH_ERR_INVALID;
  }
  LMH_CHECK_ARG(pl->units <= 0x7fffffff);
  // a launch has fewer than 2^32 threads
  int64_t most = 0;
  for (const mu_group& g : pl->groups) most += (int64_t)g.count * (g.pm / 64) * (g.pn / 64);
  LMH_CHECK_ARG(most < 0xffffff);
  if (!ws || ws_bytes < (size_t)pl->units * 256) {
    lmh_set_error("lmh_muon: workspace too small");
    return LMH_ERR_WORKSPACE;
  }
  return LMH_OK;
}

extern "C" int lmh_orthogonalize(const lmh_muon_job* jobs, int count, int dtype, int steps, float eps, void* ws, size_t ws_bytes,
                                 lmh_stream_t stream) {
  LMH_CHECK_ARG(dtype == LMH_F32 || dtype == LMH_F16 || dtype == LMH_BF16);
  mu_plan pl;
  const int rc = mu_check(jobs, count, steps, eps, ws, ws_bytes, &pl);
  if (rc != LMH_OK) return rc;
  for (int i = 0; i < count; ++i) LMH_CHECK_ARG(jobs[i].g && jobs[i].out);
  hipStream_t st = (hipStream_t)stream;
  try {
    if (dtype == LMH_F32) mu_run<f32_t, false>(jobs, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
    else if (dtype == LMH_F16) mu_run<f16_t, false>(jobs, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
    else mu_run<bf16_t, false>(jobs, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
  } catch (...) {
    lmh_set_error("lmh_orthogonalize: out of host memory");
    return LMH_ERR_INVALID;
  }
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}

extern "C" int lmh_muon_step(const lmh_muon_job* jobs, int count, int steps, float eps, float gscale, float momentum, int nesterov,
                             float lr, void* ws, size_t ws_bytes, lmh_stream_t stream) {
  mu_plan pl;
  const int rc = mu_check(jobs, count, steps, eps, ws, ws_bytes, &pl);
  if (rc != LMH_OK) return rc;
  for (int i = 0; i < count; ++i) LMH_CHECK_ARG(jobs[i].g && jobs[i].v && jobs[i].w);
  try {
    mu_run<f32_t, true>(jobs, pl, steps, eps, gscale, momentum, nesterov, lr, (char*)ws, (hipStream_t)stream);
  } catch (...) {
    lmh_set_error("lmh_muon_step: out of host memory");
    return LMH_ERR_INVALID;
  }
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}
