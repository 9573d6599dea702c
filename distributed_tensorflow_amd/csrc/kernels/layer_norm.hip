// Layer normalisation of the rows of a matrix and its gradient.
//
//   forward   mean = sum(x) / n;  var = sum((x - mean)^2) / n;  rstd = 1 / sqrt(var + eps)
//             y = (x - mean) rstd gamma + beta
//   backward  h = (x - mean) rstd;  g = dy gamma
//             dx = rstd (g - sum(g) / n - h sum(g h) / n)
//             dgamma = sum over rows of dy h;  dbeta = sum over rows of dy
//
// Both directions move every element once and do about ten operations on it: they are bound by
// memory. A row is held in registers by L lanes (a power of two from 4 to 1024, eight elements
// each), so the second look at the row that the variance needs costs no second read. Rows longer
// than 1024 lanes hold go through kernels that read them again.
//
// Everything between a load and a store is fp32. The variance is that of the differences from
// the first mean, and what those differences sum to corrects both (the "corrected two-pass"
// form): a row far from zero loses nothing but the rounding of its mean. The first mean of a
// constant row is off by the rounding of its sum, D 2^-24 of the value for sums D additions deep
// (up to 40 where the row lies in registers); the correction takes that out but for D 2^-24 of
// itself. So y is beta up to D^2 2^-48 |x| / sqrt(eps): 2e-6 for 1000 and the default epsilon.
#include "elem.h"

namespace {

enum { LN_F32 = 0, LN_BF16 = 1, LN_F16 = 2 };

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

// sum over groups of 4, 8 or 16 lanes, in every lane of the group: quads, then the halves and the
// whole of a 16-lane row by mirroring (a mirrored lane holds the other half's sum by then)
template <int L>
__device__ __forceinline__ float sum_row(float v) {
  v = dpp_add<0xB1>(v);                  // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E>(v);                  // quad_perm [2, 3, 0, 1]
  if (L >= 8) v = dpp_add<0x141>(v);     // row_half_mirror
  if (L >= 16) v = dpp_add<0x140>(v);    // row_mirror
  return v;
}

__device__ __forceinline__ float sum32(float v) {
  v = sum_row<16>(v);
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float sum64(float v) {
  v = sum32(v);
  const unsigned w = __float_as_uint(v);
  const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Sums of (a, b) over the L lanes that hold a row. L > 64: the waves' sums meet in `red` (two
// buffers of 2 * L / 64 floats per row group, used in turn: a buffer is written again only
// behind the barrier of the call in between, when every wave has read it).
template <int L>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* red, int lane, int& turn) {
  if (L <= 32) {
    a = L == 32 ? sum32(a) : sum_row<L>(a);
    b = L == 32 ? sum32(b) : sum_row<L>(b);
    return;
  }
  a = sum64(a);
  b = sum64(b);
  if (L > 64) {
    constexpr int W = L / 64;
    float* buf = red + turn * 2 * W;
    turn ^= 1;
    if ((lane & 63) == 0) {
      buf[2 * (lane >> 6)] = a;
      buf[2 * (lane >> 6) + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += buf[2 * w];
      b += buf[2 * w + 1];
    }
  }
}

constexpr int LANE_ELEMS = 8;

template <typename T>
constexpr int vec_of() {
  return 16 / (int)sizeof(T);
}

// ---- forward ------------------------------------------------------------------------------
template <typename T, typename P, int L, int NV>
__global__ __launch_bounds__(L > 256 ? L : 256) void layer_norm_kernel(
    const T* __restrict__ x, long ldx, const P* __restrict__ gamma, const P* __restrict__ beta,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, long rows,
    int cols, float eps) {
  constexpr int V = vec_of<T>();
  constexpr int BLOCK = L > 256 ? L : 256, GROUPS = BLOCK / L;
  __shared__ float red[GROUPS * 4 * (L > 64 ? L / 64 : 1)];
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  float* my_red = red + group * 4 * (L > 64 ? L / 64 : 1);
  int turn = 0;
  const float inv_n = 1.f / (float)cols;
  float gm[NV][V], bt[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (lane + j * L) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      gm[j][k] = 1.f;
      bt[j][k] = 0.f;
    }
    if (gamma) load_part<V>(gamma, c, cols, gm[j]);
    if (beta) load_part<V>(beta, c, cols, bt[j]);
  }
  // (Groups of several waves meet at barriers, so every group of a workgroup runs the same number
  // of turns; one behind the last row works on zeros. Requesting the next row before this one is
  // worked on, as the backward kernel does, made the large cases 10-25 % slower: eight or more
  // waves per SIMD cover the loads, and the registers cost some of them.)
  for (long row0 = blockIdx.x * (long)GROUPS; row0 < rows; row0 += (long)gridDim.x * GROUPS) {
    const long row = row0 + group;
    const bool live = GROUPS == 1 || row < rows;
    if (L <= 64 && !live) break;
    const T* xr = x + (live ? row : 0) * ldx;
    const int here = live ? cols : 0;
    float v[NV][V];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      load_part<V>(xr, (lane + j * L) * V, here, v[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) s += v[j][k];
    }
    group_sum2<L>(s, q, my_red, lane, turn);
    const float m0 = s / (float)cols;
    s = q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if ((j + 1) * L * V <= cols) {              // (the same for every lane)
#pragma unroll
        for (int k = 0; k < V; ++k) v[j][k] -= m0;
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          v[j][k] = (lane + j * L) * V + k < cols ? v[j][k] - m0 : 0.f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s += v[j][k];
        q = __builtin_fmaf(v[j][k], v[j][k], q);
      }
    }
    group_sum2<L>(s, q, my_red, lane, turn);
    const float fix = s * inv_n;
    const float var = __builtin_fmaf(-fix, fix, q * inv_n);
    const float rstd = 1.f / __builtin_sqrtf((var > 0.f ? var : 0.f * var) + eps);
    if (!live) continue;
    T* yr = y + row * (long)cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k)
        o[k] = __builtin_fmaf((v[j][k] - fix) * rstd, gm[j][k], bt[j][k]);
      store_part<V>(yr, (lane + j * L) * V, cols, o);
    }
    if (lane == 0 && mean_out) {
      mean_out[row] = m0 + fix;
      rstd_out[row] = rstd;
    }
  }
}

// rows longer than the registers of 1024 lanes: the same sums with the row read three times, the
// later ones in part from the L2 (bf16 4096 x 20000: 107 us, where one read and one write take 64;
// 1024 x 65536: 80 and 52; fp32 172 and 104)
template <typename T, typename P>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(
    const T* __restrict__ x, long ldx, const P* __restrict__ gamma, const P* __restrict__ beta,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, long rows,
    int cols, float eps) {
  constexpr int V = vec_of<T>(), L = 1024;
  __shared__ float red[4 * L / 64];
  const int lane = threadIdx.x;
  int turn = 0;
  const float inv_n = 1.f / (float)cols;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.f, q = 0.f, v[V];
    for (long c = lane * V; c < cols; c += L * V) {
      load_part<V>(xr, (int)c, cols, v);
#pragma unroll
      for (int k = 0; k < V; ++k) s += v[k];
    }
    group_sum2<L>(s, q, red, lane, turn);
    const float m0 = s / (float)cols;
    s = q = 0.f;
    for (long c = lane * V; c < cols; c += L * V) {
      load_part<V>(xr, (int)c, cols, v);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = c + k < cols ? v[k] - m0 : 0.f;
        s += d;
        q = __builtin_fmaf(d, d, q);
      }
    }
    group_sum2<L>(s, q, red, lane, turn);
    const float fix = s * inv_n;
    const float var = __builtin_fmaf(-fix, fix, q * inv_n);
    const float rstd = 1.f / __builtin_sqrtf((var > 0.f ? var : 0.f * var) + eps);
    T* yr = y + row * (long)cols;
    for (long c = lane * V; c < cols; c += L * V) {
      float gm[V], bt[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        gm[k] = 1.f;
        bt[k] = 0.f;
      }
      load_part<V>(xr, (int)c, cols, v);
      if (gamma) load_part<V>(gamma, (int)c, cols, gm);
      if (beta) load_part<V>(beta, (int)c, cols, bt);
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = __builtin_fmaf((v[k] - m0 - fix) * rstd, gm[k], bt[k]);
      store_part<V>(yr, (int)c, cols, v);
    }
    if (lane == 0 && mean_out) {
      mean_out[row] = m0 + fix;
      rstd_out[row] = rstd;
    }
  }
}

constexpr int grad_block(int lanes) { return lanes > 512 ? lanes : 512; }

// ---- backward -----------------------------------------------------------------------------
// Every lane adds up dy h and dy of its columns over the rows it meets; the row groups of a
// workgroup meet in LDS, the workgroups in `partial` [workgroups][2][cols] (summed in workgroup
// order by the fold kernel: no atomics, the same bits every time). A single workgroup writes
// dgamma and dbeta itself.
template <typename T, typename P, int L, int NV>
__global__ __launch_bounds__(grad_block(L)) void layer_norm_grad_kernel(
    const T* __restrict__ dy, long ldd, const T* __restrict__ x, long ldx,
    const float* __restrict__ mean, const float* __restrict__ rstd, const P* __restrict__ gamma,
    T* __restrict__ dx, float* __restrict__ partial, P* __restrict__ dgamma,
    P* __restrict__ dbeta, long rows, int cols) {
  constexpr int V = vec_of<T>();
  constexpr int BLOCK = grad_block(L), GROUPS = BLOCK / L;
  constexpr int RED = GROUPS * 4 * (L > 64 ? L / 64 : 1);
  // (rows of the fold are 64 / V words apart in banks: its readers walk along the columns)
  constexpr int FPITCH = BLOCK + 64 / V, FOLD = GROUPS > 1 ? FPITCH * 2 * V : 0;
  __shared__ float sh[RED + FOLD];
  const int group = threadIdx.x / L, lane = threadIdx.x % L;
  float* my_red = sh + group * 4 * (L > 64 ? L / 64 : 1);
  int turn = 0;
  const float inv_n = 1.f / (float)cols;
  float gm[NV][V], ag[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      gm[j][k] = 1.f;
      ag[j][k] = ab[j][k] = 0.f;
    }
    if (gamma) load_part<V>(gamma, (lane + j * L) * V, cols, gm[j]);
  }
  // Every group runs the same number of turns (L = 256: the groups share the barriers); a group
  // behind the last row works on zeros. The next row is requested before this one is
  // worked on, except with 16 elements per lane, whose registers have no room for it.
  constexpr bool AHEAD = L < 1024 || NV * V <= LANE_ELEMS;
  Pack<T, V> nx[NV], nd[NV];
  float nm = 0.f, nr = 0.f;
  auto request = [&](long row) {
    const bool live = row < rows;
    const long at = live ? row : 0;
    const int n = live ? cols : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      nx[j] = load_raw<V>(x + at * ldx, (lane + j * L) * V, n);
      nd[j] = load_raw<V>(dy + at * ldd, (lane + j * L) * V, n);
    }
    nm = live ? mean[at] : 0.f;
    nr = live ? rstd[at] : 0.f;
  };
  const long step = (long)gridDim.x * GROUPS;
  if (AHEAD) request(blockIdx.x * (long)GROUPS + group);
  for (long row0 = blockIdx.x * (long)GROUPS; row0 < rows; row0 += step) {
    const long row = row0 + group;
    if (!AHEAD) request(row);
    const float m = nm, r = nr;
    float h[NV][V], g[NV][V];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack(nx[j], h[j]);
      unpack(nd[j], g[j]);
      // (behind the row's end dy is zero, and so is everything added up here)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = g[j][k], hh = (h[j][k] - m) * r, gg = d * gm[j][k];
        ab[j][k] += d;
        ag[j][k] = __builtin_fmaf(d, hh, ag[j][k]);
        s += gg;
        q = __builtin_fmaf(gg, hh, q);
        h[j][k] = hh;
        g[j][k] = gg;
      }
    }
    if (AHEAD) request(row + step);
    group_sum2<L>(s, q, my_red, lane, turn);
    const float sn = s * inv_n, qn = q * inv_n;
    if (row < rows) {
      T* o = dx + row * (long)cols;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = r * __builtin_fmaf(-h[j][k], qn, g[j][k] - sn);
        store_part<V>(o, (lane + j * L) * V, cols, v);
      }
    }
  }
  if (!partial && !dgamma && !dbeta) return;
  float* pg = partial ? partial + blockIdx.x * 2L * cols : nullptr;
  if (GROUPS == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (lane + j * L) * V;
      if (partial) {
        store_part<V>(pg, c, cols, ag[j]);
        store_part<V>(pg + cols, c, cols, ab[j]);
      } else {
        if (dgamma) store_part<V>(dgamma, c, cols, ag[j]);
        if (dbeta) store_part<V>(dbeta, c, cols, ab[j]);
      }
    }
    return;
  }
  float* fold = sh + RED;          // [2 V][BLOCK]
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j) __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) {
      fold[k * FPITCH + threadIdx.x] = ag[j][k];
      fold[(V + k) * FPITCH + threadIdx.x] = ab[j][k];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < 2 * V * L; t += BLOCK) {
      const bool second = t >= V * L;
      const int u = second ? t - V * L : t, l = u / V, k = (second ? V : 0) + u % V;
      const int c = j * L * V + u;
      if (c >= cols) continue;
      float a = 0.f;
#pragma unroll 8
      for (int g2 = 0; g2 < GROUPS; ++g2) a += fold[k * FPITCH + g2 * L + l];
      if (partial)
        pg[(second ? cols : 0) + c] = a;
      else if (!second) {
        if (dgamma) dgamma[c] = from_f32<P>(a);
      } else if (dbeta) {
        dbeta[c] = from_f32<P>(a);
      }
    }
  }
}

// long rows: dx with two reads of the row, one workgroup per row ... (with the column sums, which
// read x and dy once more, an element per lane: bf16 4096 x 20000 243 us, where the bytes take 95;
// 1024 x 65536: 200 and 78; fp32 359 and 156)
template <typename T, typename P>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(
    const T* __restrict__ dy, long ldd, const T* __restrict__ x, long ldx,
    const float* __restrict__ mean, const float* __restrict__ rstd, const P* __restrict__ gamma,
    T* __restrict__ dx, long rows, int cols) {
  constexpr int V = vec_of<T>(), L = 1024;
  __shared__ float red[4 * L / 64];
  const int lane = threadIdx.x;
  int turn = 0;
  const float inv_n = 1.f / (float)cols;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx, *dr = dy + row * ldd;
    const float m = mean[row], r = rstd[row];
    float s = 0.f, q = 0.f, sn = 0.f, qn = 0.f;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      for (long c = lane * V; c < cols; c += L * V) {
        float v[V], d[V], gm[V];
#pragma unroll
        for (int k = 0; k < V; ++k) gm[k] = 1.f;
        load_part<V>(xr, (int)c, cols, v);
        load_part<V>(dr, (int)c, cols, d);
        if (gamma) load_part<V>(gamma, (int)c, cols, gm);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float h = c + k < cols ? (v[k] - m) * r : 0.f, g = d[k] * gm[k];
          s += g;
          q = __builtin_fmaf(g, h, q);
          v[k] = r * __builtin_fmaf(-h, qn, g - sn);
        }
        if (pass) store_part<V>(dx + row * (long)cols, (int)c, cols, v);
      }
      if (pass == 0) {
        group_sum2<L>(s, q, red, lane, turn);
        sn = s * inv_n;
        qn = q * inv_n;
      }
    }
  }
}

// ... and the column sums of one slab of rows per workgroup row (grid.y), a thread per column
template <typename T, typename P>
__global__ __launch_bounds__(256) void layer_norm_grad_cols_kernel(
    const T* __restrict__ dy, long ldd, const T* __restrict__ x, long ldx,
    const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ partial,
    long rows, int cols) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const long per = (rows + gridDim.y - 1) / gridDim.y;
  const long r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  float a = 0.f, b = 0.f;
  for (long r = r0; r < r1; ++r) {
    const float d = to_f32(dy[r * ldd + c]);
    a = __builtin_fmaf(d, (to_f32(x[r * ldx + c]) - mean[r]) * rstd[r], a);
    b += d;
  }
  float* p = partial + blockIdx.y * 2L * cols;
  p[c] = a;
  p[cols + c] = b;
}

// partial [parts][2 cols] -> dgamma, dbeta: 32 columns per workgroup, 32 threads per column each
// summing every 32nd part, then the 32 in the lanes of a wave
template <typename P>
__global__ __launch_bounds__(1024) void layer_norm_fold_kernel(const float* __restrict__ partial,
                                                               int parts, P* __restrict__ dgamma,
                                                               P* __restrict__ dbeta, int cols) {
  __shared__ float sh[32][33];
  const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
  const long c = blockIdx.x * 32L + lx;
  float a = 0.f;
  if (c < 2L * cols) {
#pragma unroll 8
    for (int p = ly; p < parts; p += 32) a += partial[p * 2L * cols + c];
  }
  sh[lx][ly] = a;
  __syncthreads();
  a = sum32(sh[ly][lx]);
  const long d = blockIdx.x * 32L + ly;
  if (lx == 0 && d < 2L * cols) {
    if (d < cols) {
      if (dgamma) dgamma[d] = from_f32<P>(a);
    } else if (dbeta) {
      dbeta[d - cols] = from_f32<P>(a);
    }
  }
}

// ---- launch -------------------------------------------------------------------------------
// (lanes, vectors per lane) for a row: eight elements per lane, 16 on 1024 lanes for the longest
// rows; lanes 0: the long-row kernels. The backward kernel keeps seven values per element (x, dy,
// gamma, the two column sums, and the next row's x and dy): with 16 elements per lane its 144
// registers left one workgroup on a CU, and 16384 x 4096 bf16 took 136 us instead of 96.
struct Plan {
  int lanes, nv;
};
Plan plan_of(long cols, int v) {
  int lanes = 4;
  while (lanes < 1024 && (long)lanes * LANE_ELEMS < cols) lanes *= 2;
  if ((long)lanes * LANE_ELEMS >= cols) return {lanes, LANE_ELEMS / v};
  if (lanes * 16L >= cols) return {lanes, 16 / v};
  return {0, 0};
}

// CALL(lanes, vectors per lane) of the plan
#define LN_FOR_PLAN(PLAN, CALL)                                       \
  if ((PLAN).nv * V > LANE_ELEMS) {                                   \
    CALL(1024, 16 / V);                                               \
  } else {                                                            \
    switch ((PLAN).lanes) {                                           \
      case 4: CALL(4, LANE_ELEMS / V); break;                         \
      case 8: CALL(8, LANE_ELEMS / V); break;                         \
      case 16: CALL(16, LANE_ELEMS / V); break;                       \
      case 32: CALL(32, LANE_ELEMS / V); break;                       \
      case 64: CALL(64, LANE_ELEMS / V); break;                       \
      case 128: CALL(128, LANE_ELEMS / V); break;                     \
      case 256: CALL(256, LANE_ELEMS / V); break;                     \
      case 512: CALL(512, LANE_ELEMS / V); break;                     \
      default: CALL(1024, LANE_ELEMS / V); break;                     \
    }                                                                 \
  }

long min_l(long a, long b) { return a < b ? a : b; }

template <typename T, typename P>
int forward(const void* x, long ldx, const void* gamma, const void* beta, void* y, float* mean,
            float* rstd, long rows, long cols, float eps, hipStream_t stream) {
  constexpr int V = vec_of<T>();
  const Plan p = plan_of(cols, V);
  if (p.lanes == 0) {
    hipLaunchKernelGGL((layer_norm_long_kernel<T, P>), dim3((unsigned)min_l(rows, 512)),
                       dim3(1024), 0, stream, (const T*)x, ldx, (const P*)gamma, (const P*)beta,
                       (T*)y, mean, rstd, rows, (int)cols, eps);
  } else {
    const int groups = p.lanes > 256 ? 1 : 256 / p.lanes;
    const long want = (rows + groups - 1) / groups;
    const dim3 grid((unsigned)min_l(want, 2048)), block(p.lanes > 256 ? p.lanes : 256);
#define LN_CALL(L_, NV_)                                                                     \
  hipLaunchKernelGGL((layer_norm_kernel<T, P, L_, NV_>), grid, block, 0, stream, (const T*)x, \
                     ldx, (const P*)gamma, (const P*)beta, (T*)y, mean, rstd, rows, (int)cols, eps)
    LN_FOR_PLAN(p, LN_CALL)
#undef LN_CALL
  }
  DTF_LAUNCH_CHECK();
  return DTF_OK;
}

// Workgroups of the backward kernel. Each turn of one takes about 1.4 us (a row per group, the
// next one requested ahead), and each leaves 2 cols sums that are written and read again: 16 cols
// bytes at 4 TB/s. The total is least at sqrt(turns * 350000 / cols) of them; up to four turns are
// left to a single workgroup, which writes the result itself.
int grad_parts(long rows, long cols, int v) {
  const Plan p = plan_of(cols, v);
  if (p.lanes == 0) return (int)min_l((rows + 15) / 16 > 0 ? (rows + 15) / 16 : 1, 64);
  const int groups = grad_block(p.lanes) / p.lanes;
  const long turns = (rows + groups - 1) / groups;
  if (turns <= 4) return 1;
  long best = (long)__builtin_sqrt((double)turns * 350000.0 / (double)cols);
  best = min_l(best < 2 ? 2 : best, grad_block(p.lanes) > 512 ? 256 : 512);
  const long each = (turns + best - 1) / best;
  return (int)((turns + each - 1) / each);
}

template <typename T, typename P>
int backward(const void* dy, long ldd, const void* x, long ldx, const float* mean,
             const float* rstd, const void* gamma, void* dx, float* partial, void* dgamma,
             void* dbeta, long rows, long cols, hipStream_t stream) {
  constexpr int V = vec_of<T>();
  const Plan p = plan_of(cols, V);
  const bool sums = dgamma || dbeta;
  const int parts = grad_parts(rows, cols, V);
  if (p.lanes == 0) {
    if (rows > 0)
      hipLaunchKernelGGL((layer_norm_grad_long_kernel<T, P>), dim3((unsigned)min_l(rows, 512)),
                         dim3(1024), 0, stream, (const T*)dy, ldd, (const T*)x, ldx, mean, rstd,
                         (const P*)gamma, (T*)dx, rows, (int)cols);
    DTF_LAUNCH_CHECK();
    if (sums)
      hipLaunchKernelGGL((layer_norm_grad_cols_kernel<T, P>),
                         dim3((unsigned)((cols + 255) / 256), parts), dim3(256), 0, stream,
                         (const T*)dy, ldd, (const T*)x, ldx, mean, rstd, partial, rows,
                         (int)cols);
  } else {
    const dim3 grid(parts), block(grad_block(p.lanes));
    const bool direct = parts == 1;
    float* part = sums && !direct ? partial : nullptr;
    P *dg = direct ? (P*)dgamma : nullptr, *db = direct ? (P*)dbeta : nullptr;
#define LN_CALL(L_, NV_)                                                                      \
  hipLaunchKernelGGL((layer_norm_grad_kernel<T, P, L_, NV_>), grid, block, 0, stream,         \
                     (const T*)dy, ldd, (const T*)x, ldx, mean, rstd, (const P*)gamma, (T*)dx, \
                     part, dg, db, rows, (int)cols)
    LN_FOR_PLAN(p, LN_CALL)
#undef LN_CALL
    if (direct) {
      DTF_LAUNCH_CHECK();
      return DTF_OK;
    }
  }
  DTF_LAUNCH_CHECK();
  if (sums) {
    hipLaunchKernelGGL((layer_norm_fold_kernel<P>), dim3((unsigned)((2 * cols + 31) / 32)),
                       dim3(1024), 0, stream, partial, parts, (P*)dgamma, (P*)dbeta, (int)cols);
    DTF_LAUNCH_CHECK();
  }
  return DTF_OK;
}

constexpr long LN_MAX_COLS = 1L << 30;

bool bad_types(int xt, int pt) {
  return xt < LN_F32 || xt > LN_F16 || (pt != xt && pt != LN_F32);
}

}  // namespace

#define LN_DISPATCH(FN, ...)                                          \
  switch (x_type * 4 + p_type) {                                      \
    case LN_F32 * 4 + LN_F32: return FN<float, float>(__VA_ARGS__);   \
    case LN_BF16 * 4 + LN_F32: return FN<dtf_bf16, float>(__VA_ARGS__); \
    case LN_BF16 * 4 + LN_BF16: return FN<dtf_bf16, dtf_bf16>(__VA_ARGS__); \
    case LN_F16 * 4 + LN_F32: return FN<_Float16, float>(__VA_ARGS__);  \
    default: return FN<_Float16, _Float16>(__VA_ARGS__);              \
  }

// y [rows, cols] (contiguous) = layer norm of x [rows, cols] (row pitch ldx elements). Types: 0
// fp32, 1 bf16, 2 fp16; p_type (gamma, beta) is x_type or fp32. gamma / beta may be null (1 / 0);
// mean / rstd: fp32 [rows], both or neither.
DTF_API int dtf_layer_norm(const void* x, long ldx, int x_type, const void* gamma,
                           const void* beta, int p_type, void* y, float* mean, float* rstd,
                           long rows, long cols, float eps, hipStream_t stream) {
  if (bad_types(x_type, p_type) || rows < 0 || cols < 1 || cols > LN_MAX_COLS ||
      (rows > 1 && ldx < cols) || !(eps >= 0.f) || (mean != nullptr) != (rstd != nullptr))
    return DTF_ERR_BAD_ARG;
  if (rows == 0) return DTF_OK;
  if (!x || !y) return DTF_ERR_BAD_ARG;
  LN_DISPATCH(forward, x, ldx, gamma, beta, y, mean, rstd, rows, cols, eps, stream)
}

// fp32 words of workspace that dtf_layer_norm_grad needs for dgamma / dbeta
DTF_API long dtf_layer_norm_grad_workspace(long rows, long cols, int x_type) {
  if (x_type < LN_F32 || x_type > LN_F16 || rows < 0 || cols < 1 || cols > LN_MAX_COLS) return 0;
  const int v = x_type == LN_F32 ? 4 : 8;
  return 2L * grad_parts(rows, cols, v) * cols;
}

// dx [rows, cols] (contiguous), dgamma [cols], dbeta [cols] (p_type; either may be null) from dy
// and x (row pitches ldd, ldx), mean, rstd [rows] and gamma (null: 1). No rows: the sums are zero.
DTF_API int dtf_layer_norm_grad(const void* dy, long ldd, const void* x, long ldx, int x_type,
                                const float* mean, const float* rstd, const void* gamma,
                                int p_type, void* dx, float* workspace, void* dgamma, void* dbeta,
                                long rows, long cols, hipStream_t stream) {
  if (bad_types(x_type, p_type) || rows < 0 || cols < 1 || cols > LN_MAX_COLS ||
      (rows > 1 && (ldx < cols || ldd < cols)))
    return DTF_ERR_BAD_ARG;
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return DTF_ERR_BAD_ARG;
  if ((dgamma || dbeta) && !workspace) return DTF_ERR_BAD_ARG;
  if (rows == 0 && !dgamma && !dbeta) return DTF_OK;
  LN_DISPATCH(backward, dy, ldd, x, ldx, mean, rstd, gamma, dx, workspace, dgamma, dbeta, rows,
              cols, stream)
}
