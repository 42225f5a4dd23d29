// Orthogonalised updates by Newton-Schulz products, for a whole list of matrices at a time (gfx950, matrix cores).
//
//   X = U / max(|U|_F, eps), taken wide (m x n, m <= n);   `steps` times:  A = X X',  X <- (a I + b A + c A A) X
//   a = 3.4445, b = -4.7750, c = 2.0315 (the published quintic: every singular value is driven to about 1)
//   optimizer:  g' = gscale g + wd w,  v = mu v + g',  U = g' + mu v (Nesterov) or v,  w -= lr scale X
//
// Arithmetic.  Small singular values grow by a = 3.44 a step, 485 times in five: 16-bit products would return noise in those
// directions, so the products have fp32 accuracy.  Every operand is held as the sum of two f16 values, hi = f16(x) and
// lo = f16(x - hi): 11 + 1 + 11 bits of x, an error of 2^-24 of its binade.  A product takes three matrix instructions (hi hi,
// hi lo, lo hi; lo lo is below 2^-24) with fp32 accumulation: 3 instead of the 6 of a bf16 split, and 2500 / 3 TFLOP/s
// against 157 of the fp32 instructions.  f16's range is enough because everything here is bounded: |X|_2 <= 1.25,
// |A| <= 1.6, |b I + c A| <= 4.8, |a I + b A + c A A| <= 3.5 (spectral norms, which bound the entries); fixed powers of two put those just below 65504, so lo keeps its
// bits down to entries of 2^-24 of the bound.
//
// Layout.  An operand lies in memory as the matrix instruction takes it ("planes"): [32 rows][16 k] units of hi then lo, 64
// lanes x 16 bytes each, k units of one row block after each other.  Tiles go to LDS with lane-linear 16-byte DMA and come
// back with ds_read_b128 at lane * 16: no bank conflicts, no address arithmetic.  A result leaves the accumulators as
// planes again: with its own rows along k straight from the registers (two lane-half swaps), the other way round through
// LDS.  All three products are then row . row products.  Rows and columns are padded with zeros to whole tiles.
//
// A and the polynomial in it are symmetric: only tiles on and above the diagonal are computed.
#include <algorithm>
#include <vector>

#include "rowops.h"

#define MU_A 3.4445f
#define MU_B -4.7750f
#define MU_C 2.0315f
// scales of what is stored as f16 pairs (powers of two)
#define MU_SX 8192.f      // X, |.| <= 1.25
#define MU_SG 8192.f      // A = X X'
#define MU_SC 8192.f      // b I + c A, eigenvalues in [b, b + 1.6 c]
#define MU_SP 8192.f      // a I + b A + c A A
#define MU_MAX_GROUPS 24  // of one launch (kernel arguments: under 4 KB together)
#define MU_MAX_JOBS 48
#define MU_NORM_BLOCKS 64

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Matrices of one padded shape: their planes lie `stride` bytes apart in the workspace.
struct mu_group {
  int64_t off, stride;
  int32_t m, n, pm, pn;
  int32_t count, tall, first, splits;
  int32_t blk0, job_blocks;        // first block of the group in this launch, blocks of one matrix
};
struct mu_table {
  int32_t groups, flip, last, pad;
  mu_group g[MU_MAX_GROUPS];
};
struct mu_ptrs { const void* g; float* v; float* w; void* out; const float* factor; float wd, scale; };
struct mu_jobs { mu_ptrs p[MU_MAX_JOBS]; };

// Buffers of one matrix, in bytes from its start.
struct mu_buf { int64_t x, xt0, xt1, a, c, p, slab, norm, end; };
__host__ __device__ inline mu_buf mu_layout(const mu_group& g) {
  mu_buf b;
  const int64_t mn = (int64_t)g.pm * g.pn * 4, mm = (int64_t)g.pm * g.pm * 4;
  b.x = 0;
  b.xt0 = b.x + mn;
  b.xt1 = b.xt0 + mn;
  b.a = b.xt1 + mn;
  b.c = b.a + mm;
  b.p = b.c + mm;
  b.slab = b.p + mm;
  b.norm = b.slab + (g.splits > 1 ? g.splits * mm : 0);
  b.end = b.norm + MU_NORM_BLOCKS * (int64_t)sizeof(double);
  return b;
}

__device__ __forceinline__ int mu_find(const mu_table& t, int blk) {
  int i = 0;
  while (i + 1 < t.groups && blk >= t.g[i + 1].blk0) ++i;
  return i;
}

__device__ __forceinline__ void mu_split(float x, uint16_t* hi, uint16_t* lo) {
  const _Float16 h = (_Float16)x;
  *hi = __builtin_bit_cast(uint16_t, h);
  *lo = __builtin_bit_cast(uint16_t, (_Float16)(x - (float)h));
}

// ---- momentum and the partial sums of the squares ----------------------------------------------------------
// u: the matrix that is orthogonalised, row-major fp32 (the optimizer's; the plain call reads its input instead)
template <typename T, bool OPT>
__global__ void __launch_bounds__(256)
k_mu_norm(mu_table tab, mu_jobs jobs, char* ws, float mu, int nesterov, float gscale) {
  __shared__ double red[4];
  const int gi = mu_find(tab, blockIdx.x);
  const mu_group& g = tab.g[gi];
  const int local = blockIdx.x - g.blk0, job = local / g.job_blocks, b = local % g.job_blocks;
  const mu_ptrs& p = jobs.p[g.first + job];
  char* base = ws + g.off + job * g.stride;
  const mu_buf buf = mu_layout(g);
  float* u = (float*)(base + buf.xt1);
  const int64_t n = (int64_t)g.m * g.n;
  const float f = OPT && p.factor ? *p.factor : 1.f;
  double acc = 0.0;
  for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n; i += (int64_t)g.job_blocks * 256) {
    float x;
    if (OPT) {
      const float gp = (((const float*)p.g)[i] * gscale + p.wd * p.w[i]) * f;
      const float v = mu * p.v[i] + gp;
      p.v[i] = v;
      x = nesterov ? gp + mu * v : v;
      u[i] = x;
    } else {
      x = to_f32(((const T*)p.g)[i]);
    }
    acc += (double)x * (double)x;
  }
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0) ((double*)(base + buf.norm))[b] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- X and X' as planes --------------------------------------------------------------------------------------
// One block: 64 x 64 of the matrix as it is stored (rows x cols), padding included.
template <typename T, bool OPT>
__global__ void __launch_bounds__(256)
k_mu_planes(mu_table tab, mu_jobs jobs, char* ws, int norm_blocks, float eps) {
  __shared__ float tile[64][65];
  const int gi = mu_find(tab, blockIdx.x);
  const mu_group& g = tab.g[gi];
  const int local = blockIdx.x - g.blk0, job = local / g.job_blocks, t = local % g.job_blocks;
  char* base = ws + g.off + job * g.stride;
  const mu_buf buf = mu_layout(g);
  const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n, prow = g.tall ? g.pn : g.pm, pcol = g.tall ? g.pm : g.pn;
  const int r0 = (t / (pcol / 64)) * 64, c0 = (t % (pcol / 64)) * 64;
  const double* part = (const double*)(base + buf.norm);
  double ss = 0.0;
  for (int i = 0; i < norm_blocks; ++i) ss += part[i];
  double norm = sqrt(ss);
  if (norm < (double)eps) norm = (double)eps;            // (not a number stays one)
  const float inv = (float)((double)MU_SX / norm);
  const void* src = OPT ? (const void*)(base + buf.xt1) : jobs.p[g.first + job].g;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = i * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
    float x = 0.f;
    if (r0 + r < rows && c0 + c < cols) {
      const int64_t at = (int64_t)(r0 + r) * cols + c0 + c;
      x = OPT ? ((const float*)src)[at] : to_f32(((const T*)src)[at]);
    }
    tile[r][c] = x * inv;
  }
  __syncthreads();
  // stored rows as rows (k = stored columns): X for a wide matrix, X' for a tall one; and the other way round
  char* by_row = base + (g.tall ? buf.xt0 : buf.x);
  char* by_col = base + (g.tall ? buf.x : buf.xt0);
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
enum { MU_GRAM = 0, MU_GRAM_SPLIT = 1, MU_GRAM_JOIN = 2, MU_POLY = 3, MU_APPLY = 4, MU_LAST = 5 };

// The 32 x 32 accumulator (lane: column lane & 31, register i: row (i & 3) + 8 (i >> 2) + 4 (lane >> 5)) as planes whose rows
// are its COLUMNS and whose k are its rows: two 16-k units at `out` (+ 2048).
__device__ __forceinline__ void mu_store_cols(const float* v, char* out, int lane) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t hi[4], lo[4];                   // [q = 2u: pairs 0, 1][q = 2u + 1: pairs 0, 1]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint16_t p0, q0, p1, q1;
      mu_split(v[8 * u + 2 * j], &p0, &q0);
      mu_split(v[8 * u + 2 * j + 1], &p1, &q1);
      hi[j] = p0 | ((uint32_t)p1 << 16);
      lo[j] = q0 | ((uint32_t)q1 << 16);
    }
    // rows 8 q + 4 (lane >> 5) + 0..3: the lane halves trade so that a lane has eight successive ones
    auto a = __builtin_amdgcn_permlane32_swap(hi[0], hi[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(hi[1], hi[3], false, false);
    auto c = __builtin_amdgcn_permlane32_swap(lo[0], lo[2], false, false);
    auto d = __builtin_amdgcn_permlane32_swap(lo[1], lo[3], false, false);
    *reinterpret_cast<raw16*>(out + u * 2048 + lane * 16) = raw16{a[0], b[0], a[1], b[1]};
    *reinterpret_cast<raw16*>(out + u * 2048 + 1024 + lane * 16) = raw16{c[0], d[0], c[1], d[1]};
  }
}
// ... the other way round (rows = its rows, k = its columns): through `t`, 32 x 33 floats of this wave's LDS.
__device__ __forceinline__ void mu_store_rows(const float* v, char* out, int lane, float* t) {
  const int l31 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < 16; ++i) t[((i & 3) + 8 * (i >> 2) + 4 * h) * 33 + l31] = v[i];
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint16_t p0, q0, p1, q1;
      mu_split(t[l31 * 33 + u * 16 + h * 8 + 2 * j], &p0, &q0);
      mu_split(t[l31 * 33 + u * 16 + h * 8 + 2 * j + 1], &p1, &q1);
      hi[j] = p0 | ((uint32_t)p1 << 16);
      lo[j] = q0 | ((uint32_t)q1 << 16);
    }
    *reinterpret_cast<raw16*>(out + u * 2048 + lane * 16) = raw16{hi[0], hi[1], hi[2], hi[3]};
    *reinterpret_cast<raw16*>(out + u * 2048 + 1024 + lane * 16) = raw16{lo[0], lo[1], lo[2], lo[3]};
  }
  __builtin_amdgcn_wave_barrier();
}

// One tile of (64 TW)^2 of C = L . R' (rows of L and R along k), 4 waves of (32 TW)^2.  Two stages of 32 k in LDS.
template <typename T, int TW, int MODE, bool OPT>
__global__ void __launch_bounds__(256)
k_mu_gemm(mu_table tab, mu_jobs jobs, char* ws, float lr) {
  constexpr int BT = 64 * TW, RB = 2 * TW, STAGE = RB * 4096;      // bytes of one operand's stage
  __shared__ __attribute__((aligned(16))) char smem[4 * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave >> 1, wc = wave & 1, l31 = lane & 31, h = lane >> 5;
  const int gi = mu_find(tab, blockIdx.x);
  const mu_group& g = tab.g[gi];
  const int local = blockIdx.x - g.blk0, job = local / g.job_blocks;
  int t = local % g.job_blocks;
  char* base = ws + g.off + job * g.stride;
  const mu_buf buf = mu_layout(g);
  const int tm = g.pm / BT, tri = tm * (tm + 1) / 2;
  const char* xt_in = base + (tab.flip ? buf.xt1 : buf.xt0);
  char* xt_out = base + (tab.flip ? buf.xt0 : buf.xt1);
  int split = 0, ti, tj, kunits, k0 = 0;
  const char *L, *R;
  if (MODE <= MU_POLY) {                     // symmetric: tile t of the upper triangle, row by row
    split = MODE == MU_GRAM_SPLIT ? t / tri : 0;
    t -= split * tri;
    ti = 0;
    int rest = t;
    while (rest >= tm - ti) { rest -= tm - ti; ++ti; }
    tj = ti + rest;
    if (MODE == MU_POLY) {
      L = base + buf.c;
      R = base + buf.a;
      kunits = g.pm / 16;
    } else {
      L = R = base + buf.x;
      kunits = g.pn / 16;
    }
  } else {
    // X' rows x polynomial rows; a wide matrix's last product the other way round: its lanes then run along stored rows
    const bool turn = MODE == MU_LAST && !g.tall;
    const int tn = g.pn / BT;
    ti = turn ? t % tm : t / tm;
    tj = turn ? t / tm : t % tm;
    (void)tn;
    L = turn ? base + buf.p : xt_in;
    R = turn ? xt_in : base + buf.p;
    kunits = g.pm / 16;
  }
  int stages = kunits / 2;
  if (MODE == MU_GRAM_SPLIT) {               // splits share the stages evenly
    k0 = (int)((int64_t)stages * split / g.splits);
    stages = (int)((int64_t)stages * (split + 1) / g.splits) - k0;
  }
  f32x16 acc[TW][TW];
#pragma unroll
  for (int a = 0; a < TW; ++a)
#pragma unroll
    for (int b = 0; b < TW; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

  if constexpr (MODE == MU_GRAM_JOIN) {      // the splits' partial tiles, in order
    const float* s = (const float*)(base + buf.slab) + (int64_t)t * BT * BT;
    for (int sp = 0; sp < g.splits; ++sp, s += (int64_t)tri * BT * BT)
#pragma unroll
      for (int a = 0; a < TW; ++a)
#pragma unroll
        for (int b = 0; b < TW; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 v = *reinterpret_cast<const float4*>(s + ((wave * TW + a) * TW + b) * 1024 + q * 256 + lane * 4);
            acc[a][b][4 * q] += v.x;
            acc[a][b][4 * q + 1] += v.y;
            acc[a][b][4 * q + 2] += v.z;
            acc[a][b][4 * q + 3] += v.w;
          }
  } else {
    typedef __attribute__((address_space(3))) void* lds_ptr;
    typedef const __attribute__((address_space(1))) void* glb_ptr;
    // a stage: RB row blocks x (2 units x 2 KB) of each operand; wave w brings in KBs w, w + 4, ...
    auto issue = [&](int s, int b) {
      char* dst = smem + b * 2 * STAGE;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int kb = i * 4 + wave;         // 1 KB piece: row block kb / 4, byte (kb % 4) KB of its stage
        const int64_t at = (int64_t)(kb >> 2) * kunits * 2048 + (int64_t)(k0 + s) * 4096 + (kb & 3) * 1024 + lane * 16;
        __builtin_amdgcn_global_load_lds((glb_ptr)(L + (int64_t)ti * RB * kunits * 2048 + at), (lds_ptr)(dst + kb * 1024), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((glb_ptr)(R + (int64_t)tj * RB * kunits * 2048 + at), (lds_ptr)(dst + STAGE + kb * 1024), 16, 0, 0);
      }
    };
    issue(0, 0);
    for (int s = 0; s < stages; ++s) {
      // this wave's pieces of stage s have landed; behind the barrier everybody's have, and everybody is done with s - 1
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (s + 1 < stages) issue(s + 1, (s + 1) & 1);
      const char* Ls = smem + (s & 1) * 2 * STAGE + wr * TW * 4096 + lane * 16;
      const char* Rs = smem + (s & 1) * 2 * STAGE + STAGE + wc * TW * 4096 + lane * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f16x8 lh[TW], ll[TW], rh[TW], rl[TW];
#pragma unroll
        for (int a = 0; a < TW; ++a) {
          lh[a] = *reinterpret_cast<const f16x8*>(Ls + a * 4096 + u * 2048);
          ll[a] = *reinterpret_cast<const f16x8*>(Ls + a * 4096 + u * 2048 + 1024);
          rh[a] = *reinterpret_cast<const f16x8*>(Rs + a * 4096 + u * 2048);
          rl[a] = *reinterpret_cast<const f16x8*>(Rs + a * 4096 + u * 2048 + 1024);
        }
#pragma unroll
        for (int a = 0; a < TW; ++a)
#pragma unroll
          for (int b = 0; b < TW; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[a], rl[b], acc[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < TW; ++a)
#pragma unroll
          for (int b = 0; b < TW; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll[a], rh[b], acc[a][b], 0, 0, 0);
#pragma unroll
        for (int a = 0; a < TW; ++a)
#pragma unroll
          for (int b = 0; b < TW; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[a], rh[b], acc[a][b], 0, 0, 0);
      }
    }
  }

  if constexpr (MODE == MU_GRAM_SPLIT) {
    float* s = (float*)(base + buf.slab) + ((int64_t)split * tri + t) * BT * BT;
#pragma unroll
    for (int a = 0; a < TW; ++a)
#pragma unroll
      for (int b = 0; b < TW; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(s + ((wave * TW + a) * TW + b) * 1024 + q * 256 + lane * 4) =
              make_float4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
    return;
  }
  if constexpr (MODE == MU_LAST) {
    const mu_ptrs& p = jobs.p[g.first + job];
    const int rows = g.tall ? g.n : g.m, cols = g.tall ? g.m : g.n;
    const float scale = OPT ? lr * p.scale / (MU_SX * MU_SP) : 1.f / (MU_SX * MU_SP);
#pragma unroll
    for (int a = 0; a < TW; ++a)
#pragma unroll
      for (int b = 0; b < TW; ++b) {
        const int c = tj * BT + (wc * TW + b) * 32 + l31;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = ti * BT + (wr * TW + a) * 32 + (i & 3) + 8 * (i >> 2) + 4 * h;
          if (r < rows && c < cols) {
            const int64_t at = (int64_t)r * cols + c;
            if (OPT) p.w[at] -= scale * acc[a][b][i];
            else ((T*)p.out)[at] = from_f32<T>(scale * acc[a][b][i]);
          }
        }
      }
    return;
  }
  __syncthreads();                           // the stages' LDS is free
  float* turn = (float*)smem + wave * 32 * 33;
#pragma unroll
  for (int a = 0; a < TW; ++a)
#pragma unroll
    for (int b = 0; b < TW; ++b) {
      const int rb = ti * RB + wr * TW + a, cb = tj * RB + wc * TW + b;      // 32-blocks of the result
      float v[16], w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool diag = MODE != MU_APPLY && rb == cb && (i & 3) + 8 * (i >> 2) + 4 * h == l31;
        if (MODE == MU_APPLY) {
          v[i] = acc[a][b][i] * (1.f / MU_SP);
        } else if (MODE == MU_POLY) {
          v[i] = acc[a][b][i] * (MU_SP / (MU_SG * MU_SC)) + (diag ? MU_A * MU_SP : 0.f);
        } else {
          v[i] = acc[a][b][i] * (MU_SG / (MU_SX * MU_SX));
          w[i] = v[i] * (MU_C * MU_SC / MU_SG) + (diag ? MU_B * MU_SC : 0.f);
        }
      }
      if constexpr (MODE == MU_APPLY) {      // rows of the result: n, columns: m
        mu_store_cols(v, base + buf.x + ((int64_t)cb * (g.pn / 16) + rb * 2) * 2048, lane);
        mu_store_rows(v, xt_out + ((int64_t)rb * (g.pm / 16) + cb * 2) * 2048, lane, turn);
      } else {
        char* d0 = base + (MODE == MU_POLY ? buf.p : buf.a);
        const int64_t at = ((int64_t)cb * (g.pm / 16) + rb * 2) * 2048, mirrored = ((int64_t)rb * (g.pm / 16) + cb * 2) * 2048;
        mu_store_cols(v, d0 + at, lane);
        if (MODE != MU_POLY) mu_store_cols(w, base + buf.c + at, lane);
        if (ti != tj) {
          mu_store_rows(v, d0 + mirrored, lane, turn);
          if (MODE != MU_POLY) mu_store_rows(w, base + buf.c + mirrored, lane, turn);
        }
      }
    }
}

// ------------------------------------------------------------------------------------------------------- host ----
struct mu_plan {
  std::vector<int> order;               // the caller's jobs, sorted by shape
  std::vector<mu_group> groups;
  std::vector<int> tw;                  // of each group
  int64_t bytes;
};

static int64_t mu_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

static void mu_make_plan(const lmh_muon_job* jobs, int count, mu_plan* pl) {
  pl->order.resize(count);
  for (int i = 0; i < count; ++i) pl->order[i] = i;
  auto key = [&](int i) {
    return std::make_pair(jobs[i].rows, jobs[i].cols);
  };
  std::stable_sort(pl->order.begin(), pl->order.end(), [&](int a, int b) { return key(a) < key(b); });
  pl->groups.clear();
  pl->tw.clear();
  int64_t tiles_all = 0;
  for (int s = 0; s < count;) {
    int e = s;
    while (e < count && key(pl->order[e]) == key(pl->order[s])) ++e;
    const lmh_muon_job& j = jobs[pl->order[s]];
    mu_group g;
    memset(&g, 0, sizeof(g));
    g.tall = j.rows > j.cols;
    g.m = g.tall ? j.cols : j.rows;
    g.n = g.tall ? j.rows : j.cols;
    const int tw = g.m > 64 ? 2 : 1, bt = 64 * tw;
    g.pm = (int)mu_up(g.m, bt);
    g.pn = (int)mu_up(g.n, bt);
    g.count = e - s;
    g.first = s;
    pl->groups.push_back(g);
    pl->tw.push_back(tw);
    const int tm = g.pm / bt;
    tiles_all += (int64_t)g.count * tm * (tm + 1) / 2;
    s = e;
  }
  int64_t off = 0;
  for (size_t i = 0; i < pl->groups.size(); ++i) {
    mu_group& g = pl->groups[i];
    // the Gram products have few tiles and a long k: split it until the launch has two blocks a compute unit, 8 stages
    // (256 k) at least to a split
    int splits = 1;
    while (tiles_all * splits < 512 && g.pn / 32 / (splits * 2) >= 8 && splits < 16) splits *= 2;
    g.splits = splits;
    const mu_buf b = mu_layout(g);
    g.stride = mu_up(b.end, 256);
    g.off = off;
    off += g.stride * g.count;
  }
  pl->bytes = off;
}

static bool mu_jobs_ok(const lmh_muon_job* jobs, int count) {
  if (!jobs || count <= 0 || count > LMH_MUON_MAX_JOBS) return false;
  for (int i = 0; i < count; ++i)
    if (jobs[i].rows <= 0 || jobs[i].cols <= 0 || jobs[i].rows > LMH_MUON_MAX_DIM || jobs[i].cols > LMH_MUON_MAX_DIM) return false;
  return true;
}

extern "C" size_t lmh_muon_workspace_bytes(const lmh_muon_job* jobs, int count) {
  if (!mu_jobs_ok(jobs, count)) return 0;
  try {
    mu_plan pl;
    mu_make_plan(jobs, count, &pl);
    return (size_t)pl.bytes + 256;
  } catch (...) {
    return 0;
  }
}

template <typename T, bool OPT>
static void mu_run(const lmh_muon_job* jobs, int count, const mu_plan& pl, int steps, float eps, float gscale, float mu, int nesterov,
                   float lr, char* ws, hipStream_t st) {
  // every launch takes groups and jobs as arguments: at most MU_MAX_GROUPS groups and MU_MAX_JOBS matrices at a time
  struct range { size_t g0, g1; };
  std::vector<mu_group> groups;
  std::vector<int> tws;
  for (size_t i = 0; i < pl.groups.size(); ++i) {       // groups of more matrices than one launch holds
    mu_group g = pl.groups[i];
    for (int done = 0; done < pl.groups[i].count; done += MU_MAX_JOBS) {
      g.count = std::min(MU_MAX_JOBS, pl.groups[i].count - done);
      g.off = pl.groups[i].off + (int64_t)done * g.stride;
      g.first = pl.groups[i].first + done;
      groups.push_back(g);
      tws.push_back(pl.tw[i]);
    }
  }
  std::vector<range> parts;
  for (size_t i = 0; i < groups.size();) {
    size_t e = i;
    int n = 0;
    while (e < groups.size() && e - i < MU_MAX_GROUPS && n + groups[e].count <= MU_MAX_JOBS) n += groups[e++].count;
    parts.push_back({i, e});
    i = e;
  }
  for (const range& r : parts) {
    mu_table tab;
    mu_jobs pj;
    memset(&tab, 0, sizeof(tab));
    memset(&pj, 0, sizeof(pj));
    const int first = groups[r.g0].first;
    int n = 0;
    for (size_t i = r.g0; i < r.g1; ++i)
      for (int k = 0; k < groups[i].count; ++k, ++n) {
        const lmh_muon_job& j = jobs[pl.order[groups[i].first + k]];
        pj.p[n] = {j.g, j.v, j.w, j.out, j.factor, j.wd, j.scale};
      }
    // blocks(g): of one matrix; tw 0: all groups
    auto fill = [&](int tw, auto blocks) {
      int total = 0, k = 0;
      for (size_t i = r.g0; i < r.g1; ++i) {
        if (tw && tws[i] != tw) continue;
        const int per = blocks(groups[i]);
        if (per == 0) continue;
        tab.g[k] = groups[i];
        tab.g[k].first -= first;
        tab.g[k].blk0 = total;
        tab.g[k].job_blocks = per;
        total += per * groups[i].count;
        ++k;
      }
      tab.groups = k;
      return total;
    };
    int nb = fill(0, [](const mu_group&) { return MU_NORM_BLOCKS; });
    lmh_launch((k_mu_norm<T, OPT>), dim3(nb), dim3(256), 0, st, tab, pj, ws, mu, nesterov, gscale);
    nb = fill(0, [](const mu_group& g) { return (g.pm / 64) * (g.pn / 64); });
    lmh_launch((k_mu_planes<T, OPT>), dim3(nb), dim3(256), 0, st, tab, pj, ws, MU_NORM_BLOCKS, eps);
#define MU_GEMM(MODE_, BLOCKS_)                                                                                \
  do {                                                                                                         \
    for (int tw = 1; tw <= 2; ++tw) {                                                                          \
      const int bt = 64 * tw;                                                                                  \
      nb = fill(tw, [&](const mu_group& g) { const int tm = g.pm / bt, tri = tm * (tm + 1) / 2, tn = g.pn / bt; (void)tri; (void)tn; return (BLOCKS_); }); \
      if (nb == 0) continue;                                                                                   \
      if (tw == 1) lmh_launch((k_mu_gemm<T, 1, MODE_, OPT>), dim3(nb), dim3(256), 0, st, tab, pj, ws, lr);     \
      else lmh_launch((k_mu_gemm<T, 2, MODE_, OPT>), dim3(nb), dim3(256), 0, st, tab, pj, ws, lr);             \
    }                                                                                                          \
  } while (0)
    for (int it = 0; it < steps; ++it) {
      tab.flip = it & 1;
      MU_GEMM(MU_GRAM, (g.splits == 1 ? tri : 0));
      MU_GEMM(MU_GRAM_SPLIT, (g.splits > 1 ? tri * g.splits : 0));
      MU_GEMM(MU_GRAM_JOIN, (g.splits > 1 ? tri : 0));
      MU_GEMM(MU_POLY, tri);
      if (it + 1 < steps) MU_GEMM(MU_APPLY, tm * tn);
      else MU_GEMM(MU_LAST, tm * tn);
    }
#undef MU_GEMM
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
  if (!ws || ws_bytes < (size_t)pl->bytes) {
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
    if (dtype == LMH_F32) mu_run<f32_t, false>(jobs, count, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
    else if (dtype == LMH_F16) mu_run<f16_t, false>(jobs, count, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
    else mu_run<bf16_t, false>(jobs, count, pl, steps, eps, 1.f, 0.f, 0, 0.f, (char*)ws, st);
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
    mu_run<f32_t, true>(jobs, count, pl, steps, eps, gscale, momentum, nesterov, lr, (char*)ws, (hipStream_t)stream);
  } catch (...) {
    lmh_set_error("lmh_muon_step: out of host memory");
    return LMH_ERR_INVALID;
  }
  LMH_CHECK_LAUNCH();
  return LMH_OK;
}
