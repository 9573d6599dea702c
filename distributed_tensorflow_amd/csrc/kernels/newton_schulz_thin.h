// Newton-Schulz orthogonalisation of matrices with m = min(rows, cols) <= 64 (included by
// newton_schulz.hip, whose descriptors it uses).
//
// X only ever meets polynomials of X X^T, so for few rows the steps need X at their ends only:
//
//   A = X X^T  (m x m);   per step:  B = a I + b A + c A A,  Q = Q B,  A = B A B;   X = Q X
//
// The tiled sequence spends its time on launches here (2 + 3 steps of them, 6.4 us each); this
// form takes two -- the sums A over the columns, then everything else -- or one for n <= 256.
// A holds the squares of the singular values, and a direction of size s relative to the largest
// would be off by 2^-24 / s^2 in fp32: all of it is done in 64 bits, on the fp64 matrix
// instruction (the bound: 17 products of 64^3 take 12 us of one CU), and the result is rounded
// once. All matrices are symmetric and commute: one triangle of 16 x 16 tiles is computed, and
// an operand is read by rows whichever side it stands on.
//
// Every workgroup of the second launch adds up the same partial sums and goes through the same
// polynomials by itself before it multiplies its own columns.
#pragma once

constexpr int THIN_M = 64;
constexpr int THIN_THREADS = 512, THIN_WAVES = 8;
constexpr int THIN_GRAM = 10 * 256;        // doubles of a slab's sums: 10 lower tiles
constexpr int THIN_ONE = 256;              // columns up to which one workgroup does it all
constexpr int THIN_COLS = 16 * THIN_WAVES; // columns a workgroup multiplies at a time

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct NsSteps {
  float c[3 * NS_MAX_STEPS];
  int steps;
};

// Workgroups that share the sums over n columns. A wave takes 8 ns per column of its slab's
// share, the second launch 0.35 us per slab to add: their sum is least near sqrt(n / 40).
inline long thin_slabs(long n) {
  if (n <= THIN_ONE) return 1;
  long s = 1;
  while (s * s * 32 < n) ++s;
  return s;
}

__device__ __forceinline__ f64x4 mfma64(double a, double b, f64x4 c) {
  return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// lower tiles in the order (0,0) (1,0) (1,1) (2,0) ...
__device__ __forceinline__ void tile_at(int tile, int& ti, int& tj) {
  ti = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0;
  tj = tile - ti * (ti + 1) / 2;
}

// Sums of X X^T over columns [begin, end) in the accumulators of wave 0. A lane of the matrix
// instruction holds row l % 16 of a block at column l / 16, on either side, so one register
// serves both. ADVANCE: the momentum is advanced on the way (every element passes here once).
template <typename E, bool ADVANCE, int MT>
__device__ __forceinline__ void thin_gram(const NsMat& t, const NsMuon& mo, int begin, int end,
                                          f64x4 (&acc)[MT * (MT + 1) / 2], double* red) {
  constexpr int TILES = MT * (MT + 1) / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane & 15, q = lane >> 4;
  const bool tall = t.rows > t.cols;
  const E* g = (const E*)t.g;
#pragma unroll
  for (int k = 0; k < TILES; ++k) acc[k] = f64x4{0.0, 0.0, 0.0, 0.0};
  for (int c0 = begin + 16 * wave; c0 < end; c0 += 16 * THIN_WAVES) {
    float u[MT][4];
#pragma unroll
    for (int b = 0; b < MT; ++b) {
      const int i = 16 * b + row;
      if (!tall) {
        const int stop = i < t.m ? end : 0, c = c0 + 4 * q;
        const long at = i < t.m ? (long)i * t.n : 0;
        load_part<4>(g + at, c, stop, u[b]);
        if (ADVANCE) {
          float v[4];
          load_part<4>(t.v + at, c, stop, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = __builtin_fmaf(mo.mu, v[k], u[b][k]);
            u[b][k] = mo.nesterov ? __builtin_fmaf(mo.mu, v[k], u[b][k]) : v[k];
          }
          store_part<4>(t.v + at, c, stop, v);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = c0 + 4 * k + q;
          u[b][k] = 0.f;
          if (i < t.m && c < end) {
            const long at = (long)c * t.m + i;
            u[b][k] = to_f32(g[at]);
            if (ADVANCE) {
              const float v = __builtin_fmaf(mo.mu, t.v[at], u[b][k]);
              t.v[at] = v;
              u[b][k] = mo.nesterov ? __builtin_fmaf(mo.mu, v, u[b][k]) : v;
            }
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int ti = 0; ti < MT; ++ti)
#pragma unroll
        for (int tj = 0; tj <= ti; ++tj)
          acc[ti * (ti + 1) / 2 + tj] =
              mfma64((double)u[ti][k], (double)u[tj][k], acc[ti * (ti + 1) / 2 + tj]);
  }
  // the waves' sums, by halves
#pragma unroll
  for (int half = THIN_WAVES / 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      double* mine = red + (wave - half) * TILES * 256;
#pragma unroll
      for (int k = 0; k < TILES; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) mine[k * 256 + r * 64 + lane] = acc[k][r];
    }
    __syncthreads();
    if (wave < half) {
      const double* theirs = red + wave * TILES * 256;
#pragma unroll
      for (int k = 0; k < TILES; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[k][r] += theirs[k * 256 + r * 64 + lane];
    }
    __syncthreads();
  }
}

// One symmetric product P R of the matrices in LDS: this wave's tiles (wave, wave + 8)
template <int MT>
__device__ __forceinline__ void thin_product(const double* P, const double* R, f64x4 (&out)[2]) {
  constexpr int TILES = MT * (MT + 1) / 2, PITCH = 16 * MT + 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int tile = wave + 8 * s;
    if (tile >= TILES) continue;
    int ti, tj;
    tile_at(tile, ti, tj);
    const double* p = P + (16 * ti + (lane & 15)) * PITCH + (lane >> 4);
    const double* r = R + (16 * tj + (lane & 15)) * PITCH + (lane >> 4);
    f64x4 even = {0.0, 0.0, 0.0, 0.0}, odd = {0.0, 0.0, 0.0, 0.0};   // two chains: half the wait
#pragma unroll 4
    for (int k = 0; k < 16 * MT; k += 8) {
      even = mfma64(p[k], r[k], even);
      odd = mfma64(p[k + 4], r[k + 4], odd);
    }
    out[s] = even + odd;
  }
}

// F(value, i, j) of every element of this wave's tiles, written to both places
template <int MT, typename F>
__device__ __forceinline__ void thin_store(double* to, const f64x4 (&v)[2], F&& f) {
  constexpr int TILES = MT * (MT + 1) / 2, PITCH = 16 * MT + 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int tile = wave + 8 * s;
    if (tile >= TILES) continue;
    int ti, tj;
    tile_at(tile, ti, tj);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * ti + 4 * r + (lane >> 4), j = 16 * tj + (lane & 15);
      const double x = f(v[s][r], i, j);
      to[i * PITCH + j] = x;
      if (ti != tj) to[j * PITCH + i] = x;
    }
  }
}

// A (sums, unscaled) -> Q with the norm divided out of it
template <int MT>
__device__ __forceinline__ double thin_polynomials(double* A, double* B, double* Q, int m,
                                                   const NsSteps& st, float eps) {
  constexpr int PITCH = 16 * MT + 2;
  double trace = 0.0;
  for (int i = 0; i < m; ++i) trace += A[i * PITCH + i];
  const double inv = 1.0 / (__builtin_sqrt(trace) + (double)eps), inv2 = inv * inv;
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * PITCH; i += THIN_THREADS) A[i] *= inv2;
  __syncthreads();
  for (int k = 0; k < st.steps; ++k) {
    const double a = st.c[3 * k], b = st.c[3 * k + 1], c = st.c[3 * k + 2];
    f64x4 v[2], w[2];
    thin_product<MT>(A, A, v);
    auto poly = [&](double x, int i, int j) {
      return __builtin_fma(c, x, __builtin_fma(b, A[i * PITCH + j], i == j ? a : 0.0));
    };
    thin_store<MT>(B, v, poly);
    if (k == 0) thin_store<MT>(Q, v, poly);
    __syncthreads();
    const bool more = k + 1 < st.steps;
    if (k > 0) thin_product<MT>(Q, B, w);
    if (more) thin_product<MT>(A, B, v);
    __syncthreads();
    auto same = [](double x, int, int) { return x; };
    if (k > 0) thin_store<MT>(Q, w, same);
    if (more) thin_store<MT>(A, v, same);
    __syncthreads();
    if (more) {
      thin_product<MT>(A, B, v);
      __syncthreads();
      thin_store<MT>(A, v, same);
      __syncthreads();
    }
  }
  return inv;
}

// columns [begin, end) of the result, 16 per wave at a time
template <typename E, bool MUON, int MT>
__device__ __forceinline__ void thin_apply(const NsMat& t, const NsMuon& mo, const double* Q,
                                           double inv, int begin, int end) {
  constexpr int PITCH = 16 * MT + 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, q = lane >> 4;
  const bool tall = t.rows > t.cols;
  const float lr = MUON ? (mo.lr_dev ? mo.lr_dev[0] : mo.lr) : 0.f;
  const float keep = 1.f - lr * mo.decay, take = lr * t.scale;
  E* out = (E*)t.out;
  for (int c0 = begin + 16 * wave; c0 < end; c0 += THIN_COLS) {
    const int j = c0 + col;
    float u[4 * MT];
#pragma unroll
    for (int k = 0; k < 4 * MT; ++k) {
      const int i = 4 * k + q;
      u[k] = 0.f;
      if (i < t.m && j < end) {
        const long at = tall ? (long)j * t.m + i : (long)i * t.n + j;
        u[k] = to_f32(((const E*)t.g)[at]);
        if (MUON) {
          const float v = t.v[at];                 // already advanced
          u[k] = mo.nesterov ? __builtin_fmaf(mo.mu, v, u[k]) : v;
        }
      }
    }
    f64x4 acc[MT];
#pragma unroll
    for (int b = 0; b < MT; ++b) acc[b] = f64x4{0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < 4 * MT; ++k) {
#pragma unroll
      for (int b = 0; b < MT; ++b)
        acc[b] = mfma64(Q[(16 * b + col) * PITCH + 4 * k + q], (double)u[k], acc[b]);
      if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (all of Q in registers would spill)
    }
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * r + q;
        if (i >= t.m || j >= end) continue;
        const long at = tall ? (long)j * t.m + i : (long)i * t.n + j;
        const float o = (float)(acc[b][r] * inv);
        if (MUON) {
          float* w = (float*)t.out;
          w[at] = __builtin_fmaf(-take, o, keep * w[at]);
        } else {
          out[at] = from_f32<E>(o);
        }
      }
  }
}

template <int MT>
constexpr int thin_lds() {
  constexpr int poly = 3 * 16 * MT * (16 * MT + 2) * 8;
  constexpr int red = THIN_WAVES / 2 * (MT * (MT + 1) / 2) * 256 * 8;
  return poly > red ? poly : red;
}

// first launch: a workgroup per slab
template <typename E, bool MUON, int MT>
__global__ __launch_bounds__(THIN_THREADS) void ns_thin_gram_kernel(NsArgs args, NsMuon mo) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int TILES = MT * (MT + 1) / 2;
  const NsMat& t = args.t[matrix_of(args, blockIdx.x)];
  const int slab = blockIdx.x - args.first[matrix_of(args, blockIdx.x)];
  const int begin = slab * t.slab_cols;
  const int end = begin + t.slab_cols < t.n ? begin + t.slab_cols : t.n;
  f64x4 acc[TILES];
  thin_gram<E, MUON, MT>(t, mo, begin, end, acc, (double*)smem);
  if (threadIdx.x < 64) {
    double* to = t.gram + (long)slab * THIN_GRAM + threadIdx.x;
#pragma unroll
    for (int k = 0; k < TILES; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) to[k * 256 + r * 64] = acc[k][r];
  }
}

// second launch, a workgroup per block of columns; ONE: the only launch, a workgroup per matrix
template <typename E, bool MUON, int MT, bool ONE>
__global__ __launch_bounds__(THIN_THREADS) void ns_thin_apply_kernel(NsArgs args, NsSteps st,
                                                                     float eps, NsMuon mo) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int TILES = MT * (MT + 1) / 2, PITCH = 16 * MT + 2, SIZE = 16 * MT * PITCH;
  double *A = (double*)smem, *B = A + SIZE, *Q = B + SIZE;
  const int mat = matrix_of(args, blockIdx.x);
  const NsMat& t = args.t[mat];
  const int block = blockIdx.x - args.first[mat], blocks = args.first[mat + 1] - args.first[mat];
  auto put = [&](int at, double x) {
    int ti, tj;
    tile_at(at >> 8, ti, tj);
    const int i = 16 * ti + 4 * ((at >> 6) & 3) + ((at & 63) >> 4), j = 16 * tj + (at & 15);
    A[i * PITCH + j] = x;
    if (ti != tj) A[j * PITCH + i] = x;
  };
  if (ONE) {
    f64x4 acc[TILES];
    thin_gram<E, MUON, MT>(t, mo, 0, t.n, acc, (double*)smem);
    if (threadIdx.x < 64) {
#pragma unroll
      for (int k = 0; k < TILES; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) put(k * 256 + r * 64 + threadIdx.x, acc[k][r]);
    }
  } else {
    for (int at = threadIdx.x; at < TILES * 256; at += THIN_THREADS) {
      double x = 0.0;
#pragma unroll 4
      for (int s = 0; s < t.slabs; ++s) x += t.gram[(long)s * THIN_GRAM + at];
      put(at, x);
    }
  }
  __syncthreads();
  const double inv = thin_polynomials<MT>(A, B, Q, t.m, st, eps);
  const int per = (t.n + blocks - 1) / blocks + 15 & ~15;
  const int begin = block * per, end = begin + per < t.n ? begin + per : t.n;
  thin_apply<E, MUON, MT>(t, mo, Q, inv, begin, end);
}

template <typename KernelT>
void allow_lds(KernelT kernel, int lds) {
  (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename E, bool MUON, int MT>
int launch_thin_of(NsArgs args, const NsSteps& st, float eps, const NsMuon& mo,
                   hipStream_t stream) {
  constexpr int LDS = thin_lds<MT>();
  static DtfPerDeviceOnce once;
  dtf_once_per_device(once, [&] {
    allow_lds(ns_thin_gram_kernel<E, MUON, MT>, LDS);
    allow_lds(ns_thin_apply_kernel<E, MUON, MT, false>, LDS);
    allow_lds(ns_thin_apply_kernel<E, MUON, MT, true>, LDS);
  });
  const dim3 threads(THIN_THREADS);
  bool one = true;
  for (int i = 0; i < args.count; ++i) one = one && args.t[i].n <= THIN_ONE;
  if (one) {
    for (int i = 0; i < args.count; ++i) args.first[i + 1] = i + 1;
    hipLaunchKernelGGL((ns_thin_apply_kernel<E, MUON, MT, true>), dim3(args.count), threads, LDS,
                       stream, args, st, eps, mo);
    DTF_LAUNCH_CHECK();
    return DTF_OK;
  }
  for (int i = 0; i < args.count; ++i) args.first[i + 1] = args.first[i] + args.t[i].slabs;
  hipLaunchKernelGGL((ns_thin_gram_kernel<E, MUON, MT>), dim3(args.first[args.count]), threads, LDS,
                     stream, args, mo);
  DTF_LAUNCH_CHECK();
  for (int i = 0; i < args.count; ++i) {
    const int blocks = (args.t[i].n + THIN_COLS - 1) / THIN_COLS;
    args.first[i + 1] = args.first[i] + (blocks < 512 ? blocks : 512);
  }
  hipLaunchKernelGGL((ns_thin_apply_kernel<E, MUON, MT, false>), dim3(args.first[args.count]),
                     threads, LDS, stream, args, st, eps, mo);
  DTF_LAUNCH_CHECK();
  return DTF_OK;
}

template <typename E, bool MUON>
int launch_thin(const NsArgs& args, int steps, const float* coef, float eps, const NsMuon& mo,
                hipStream_t stream) {
  NsSteps st = {};
  st.steps = steps;
  for (int k = 0; k < 3 * steps; ++k) st.c[k] = coef[k];
  int m = 1;
  for (int i = 0; i < args.count; ++i) m = args.t[i].m > m ? args.t[i].m : m;
  // (blocks of 16 rows beyond a matrix's own hold zeros: they change no bit of its result)
  if (m <= 16) return launch_thin_of<E, MUON, 1>(args, st, eps, mo, stream);
  if (m <= 32) return launch_thin_of<E, MUON, 2>(args, st, eps, mo, stream);
  if (m <= 48) return launch_thin_of<E, MUON, 3>(args, st, eps, mo, stream);
  return launch_thin_of<E, MUON, 4>(args, st, eps, mo, stream);
}
