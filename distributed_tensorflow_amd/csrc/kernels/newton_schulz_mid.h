// Newton-Schulz orthogonalisation of matrices with 64 < m <= 128 rows and n <= 2048 columns (m =
// min(rows, cols); included by newton_schulz.hip, whose descriptors and images it uses).
//
// The tiled sequence takes three launches a step of about 6 us each here, with almost nothing in
// them. An m x m matrix as fp16 pairs is 64 KB, so two of them fit a workgroup, and a slab of 128
// columns of X in place of one: every workgroup adds up A = X X^T from the slabs' parts, goes
// through the polynomials of one step or of a pair of them by itself, multiplies its own slab, X =
// P X, and leaves the slab's part of the next A. Five steps are five launches with the norm and the
// first A: 128 x 128 64 us (tiled 86), 784 x 100 77 (105), 128 x 2048 93 (111), sixteen 128 x 2048 145
// (163). A slab costs 0.7 us a launch to add up, so rows longer than 2048 are left to the tiles, and
// so are calls with a larger matrix, whose launches take these along.
//
// What bounds it: 2 to 3 us a product on one CU, of which the matrix instructions are 1.3 and the
// LDS reads as much; the rest is rounding to pairs and two barriers.
//
// One buffer holds B, the other A, then C = B A, A' = C B, B' = q'(A'), and P = B' B goes where B
// was. The products are commuting polynomials of one A, symmetric up to rounding, and are read by
// rows on either side. Sums over 128 elements at most run in one accumulator, as in the tiles.
#pragma once

constexpr int MID_M = 128, MID_N = 2048, MID_SLAB = 128;
constexpr int MID_THREADS = 512;
constexpr int MID_KT = MID_M * 128;                    // bytes of a K-tile of 32: 128 rows
constexpr int MID_MAT = 4 * MID_KT;                    // of a matrix of pairs
constexpr int MID_PART = MID_M * MID_SLAB * 4;         // of a slab's part of A

struct MidArgs {
  NsMat t[NS_MAX_MATS];
  int first[NS_MAX_MATS + 1];
  int count;
  int pair;                      // two steps in this launch
  int turn;                      // launches before this one: which parts are read
  float c[6];                    // (a, b, c) of the steps
};

// Rows m0 .. + 63, columns n0 .. + 31 of P Q^T over KT K-tiles
template <int KT>
__device__ __forceinline__ void mid_product(const char* P, const char* Q, int m0, int n0,
                                            f32x4 (&acc)[4][2]) {
  const int lane = threadIdx.x & 63, frow = lane & 15, fq = lane >> 4;
  f32x4 cross[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = cross[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    f16x8 ph[4], pl[4], qh[2], ql[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* at = Q + kt * MID_KT;
      qh[j] = *reinterpret_cast<const f16x8*>(at + piece_off(n0 + 16 * j + frow, fq));
      ql[j] = *reinterpret_cast<const f16x8*>(at + piece_off(n0 + 16 * j + frow, 4 + fq));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* at = P + kt * MID_KT;
      ph[i] = *reinterpret_cast<const f16x8*>(at + piece_off(m0 + 16 * i + frow, fq));
      pl[i] = *reinterpret_cast<const f16x8*>(at + piece_off(m0 + 16 * i + frow, 4 + fq));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // (operands swapped: a lane's four results lie along the columns)
        cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[j], ph[i], cross[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[j], ph[i], acc[i][j], 0, 0, 0);
        cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[j], pl[i], cross[i][j], 0, 0, 0);
      }
  }
  add_cross(acc, cross);
}

// byte offset of elements n .. n + 3 of row m (hi; n a multiple of four) in a matrix of pairs
__device__ __forceinline__ int mid_off(int m, int n, int lo) {
  return (n >> 5) * MID_KT + piece_off(m, 4 * lo + ((n & 31) >> 3)) + (n & 7) * 2;
}

__device__ __forceinline__ void mid_put(char* to, int m, int n, f32x4 v) {
  uint2 hi, lo;
  split4(v, hi, lo);
  *reinterpret_cast<uint2*>(to + mid_off(m, n, 0)) = hi;
  *reinterpret_cast<uint2*>(to + mid_off(m, n, 1)) = lo;
}

// rows r0 .. of an image of `rows` rows and kts K-tiles -> LDS; what is not there becomes zeros
__device__ __forceinline__ void mid_request(const char* image, int rows, int r0, int kts,
                                            u32x4 (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int piece = k * MID_THREADS + threadIdx.x;       // [4 K-tiles][128 rows][8]
    const int kt = piece >> 10, row = (piece >> 3) & 127, kc = piece & 7;
    v[k] = u32x4{0, 0, 0, 0};
    if (r0 + row < rows && kt < kts)
      v[k] = *reinterpret_cast<const u32x4*>(image + image_off(rows, r0 + row, 32 * kt) + kc * 16);
  }
}
__device__ __forceinline__ void mid_land(char* to, const u32x4 (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int piece = k * MID_THREADS + threadIdx.x;
    const int kt = piece >> 10, row = (piece >> 3) & 127, kc = piece & 7;
    *reinterpret_cast<u32x4*>(to + kt * MID_KT + piece_off(row, kc)) = v[k];
  }
}

// MID_FIRST: X from G, and its A. MID_STEP: one or two steps. MID_LAST: these, to the caller's
// matrix
enum { MID_FIRST, MID_STEP, MID_LAST };

template <int KT, typename E, int WHERE, bool MUON>
__global__ __launch_bounds__(MID_THREADS) void ns_mid_kernel(MidArgs args, float eps, NsMuon mo) {
  constexpr bool LAST = WHERE == MID_LAST;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char *U = smem, *V = smem + MID_MAT;
  int mat = 0;
  while (mat + 1 < args.count && (int)blockIdx.x >= args.first[mat + 1]) ++mat;
  const NsMat& t = args.t[mat];
  const int slab = blockIdx.x - args.first[mat], slabs = args.first[mat + 1] - args.first[mat];
  const int n0 = slab * MID_SLAB, width = t.n - n0 < MID_SLAB ? t.n - n0 : MID_SLAB;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 15, fq = lane >> 4;
  const int wm = (wave >> 2) * 64, wn = (wave & 3) * 32;
  const bool tall = t.rows > t.cols;
  f32x4 acc[4][2];
  auto each = [&](auto&& f) {                    // f(i, j, row, first of four columns)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) f(i, j, wm + 16 * i + frow, wn + 16 * j + 4 * fq);
  };
  if constexpr (WHERE == MID_FIRST) {
    double sum = 0.0;
    for (int p = threadIdx.x; p < t.nparts; p += MID_THREADS) sum += t.parts[p];
    const E* g = (const E*)t.g;
    each([&](int i, int j, int m, int n) {
      float u[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
      if (!tall) {
        const long at = m < t.m ? (long)m * t.n : 0;
        const int stop = m < t.m ? t.n : 0;
        load_part<4>(g + at, n0 + n, stop, u);
        if (MUON) load_part<4>(t.v + at, n0 + n, stop, v);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m < t.m && n + r < width) {
            const long at = (long)(n0 + n + r) * t.m + m;
            u[r] = to_f32(g[at]);
            if (MUON) v[r] = t.v[at];
          }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)                // (the momentum is already advanced)
        acc[i][j][r] = MUON ? mo.nesterov ? __builtin_fmaf(mo.mu, v[r], u[r]) : v[r] : u[r];
    });
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    double* sums = (double*)V;
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < MID_THREADS / 64; ++k) sum += sums[k];
    // (the quotient is taken in 64 bits as well: a norm may lie beyond fp32's range)
    const double mul = (double)X_SCALE / (__builtin_sqrt(sum) + (double)eps);
    each([&](int i, int j, int m, int n) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        // (0 / 0 of a zero matrix without epsilon stays in the matrix: padding is zero always)
        acc[i][j][r] = m < t.m && n + r < width ? (float)((double)acc[i][j][r] * mul) : 0.f;
    });
  } else {
    u32x4 held[8];
    mid_request(t.xt0, t.n, n0, t.km / 32, held);
    // A: the parts in slab order
    const __amdgpu_buffer_rsrc_t parts = __builtin_amdgcn_make_buffer_rsrc(
        (void*)t.a_parts[(args.turn + 1) & 1], 0, slabs * MID_PART, 0x00020000);
    // (16 x 16 blocks behind the last row or column are not fetched: an offset out of range)
    int at[4][2];
    each([&](int i, int j, int, int) {
      acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      at[i][j] = wm + 16 * i < t.m && wn + 16 * j < t.m
                     ? ((i * 2 + j) * MID_THREADS + (int)threadIdx.x) * 16
                     : 0x40000000;
    });
#pragma unroll 4
    for (int s = 0; s < slabs; ++s) {
      f32x4 v[4][2];
      each([&](int i, int j, int, int) {
        v[i][j] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, at[i][j], s * MID_PART, 0));
      });
      each([&](int i, int j, int, int) { acc[i][j] += v[i][j]; });
    }
    each([&](int i, int j, int m, int n) {
      mid_put(U, m, n, acc[i][j] * (AB_SCALE / (X_SCALE * X_SCALE)));
    });
    __syncthreads();
    // a I + b A + c A A of the A in U
    auto polynomial = [&](const float* c) {
      mid_product<KT>(U, U, wm, wn, acc);
      each([&](int i, int j, int m, int n) {
        const f16x4 hi = *reinterpret_cast<const f16x4*>(U + mid_off(m, n, 0));
        const f16x4 lo = *reinterpret_cast<const f16x4*>(U + mid_off(m, n, 1));
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][j][r] = __builtin_fmaf(
              c[2] / AB_SCALE, acc[i][j][r],
              __builtin_fmaf(c[1], joined(hi[r], lo[r]),
                             m == n + r && m < t.m ? c[0] * AB_SCALE : 0.f));
      });
    };
    auto put = [&](char* to, float mul) {
      each([&](int i, int j, int m, int n) { mid_put(to, m, n, acc[i][j] * mul); });
      __syncthreads();
    };
    polynomial(args.c);
    put(V, 1.f);                                 // B
    if (args.pair) {
      mid_product<KT>(V, U, wm, wn, acc);
      __syncthreads();
      put(U, 1.f / AB_SCALE);                    // C = B A
      mid_product<KT>(U, V, wm, wn, acc);
      __syncthreads();
      put(U, 1.f / AB_SCALE);                    // A' = C B
      polynomial(args.c + 3);
      __syncthreads();
      put(U, 1.f);                               // B'
      mid_product<KT>(U, V, wm, wn, acc);
      __syncthreads();
      put(V, 1.f / AB_SCALE);                    // P = B' B
    }
    // (behind the last barrier nobody reads U)
    mid_land(U, held);
    __syncthreads();
    if (LAST && tall)                            // the result as the caller lays it
      mid_product<KT>(U, V, wm, wn, acc);
    else
      mid_product<KT>(V, U, wm, wn, acc);
    if constexpr (LAST) {
      const float lr = MUON ? (mo.lr_dev ? mo.lr_dev[0] : mo.lr) : 0.f;
      const float keep = 1.f - lr * mo.decay, take = lr * t.scale;
      const int rows = tall ? width : t.m, cols = tall ? t.m : width;
      E* out = (E*)t.out + (tall ? (long)n0 * t.m : n0);
      const long ld = tall ? t.m : t.n;
      each([&](int i, int j, int m, int n) {
        if (m >= rows || n >= cols) return;
        E* row = out + m * ld;
        float v[4], old[4];
        if (MUON) load_part<4>(row, n, cols, old);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = acc[i][j][r] * (1.f / (X_SCALE * AB_SCALE));
          if (MUON) v[r] = __builtin_fmaf(-take, v[r], keep * old[r]);
        }
        store_part<4>(row, n, cols, v);
      });
      return;
    }
    each([&](int i, int j, int, int) { acc[i][j] *= 1.f / AB_SCALE; });
  }
  if constexpr (!LAST) {
    __syncthreads();                             // what was read makes place for the new X
    unsigned* strip = reinterpret_cast<unsigned*>(V) + wave * (32 * 36);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x4 v = acc[2 * h + i][j];
          mid_put(U, wm + 32 * h + 16 * i + frow, wn + 16 * j + 4 * fq, v);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            strip[(16 * j + 4 * fq + r) * 36 + 16 * i + frow] = split_pack(v[r]);
        }
      __builtin_amdgcn_wave_barrier();
      // its transpose for the next launch, through the strip: [32 columns][32 rows]
      const int m = wm + 32 * h;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int nl = 16 * q + (lane >> 2), n = wn + nl;
        unsigned p[8];
        const u32x4* src = reinterpret_cast<const u32x4*>(strip + nl * 36 + (lane & 3) * 8);
        *reinterpret_cast<u32x4*>(p) = src[0];
        *reinterpret_cast<u32x4*>(p + 4) = src[1];
        if (n < width && m < t.m)
          store_split8(t.xt0 + image_off(t.n, n0 + n, m + (lane & 3) * 8), p);
      }
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    mid_product<4>(U, U, wm, wn, acc);
    f32x4* part = reinterpret_cast<f32x4*>(t.a_parts[args.turn & 1] + (long)slab * MID_PART) +
                  threadIdx.x;
    each([&](int i, int j, int, int) {
      if (wm + 16 * i < t.m && wn + 16 * j < t.m) part[(i * 2 + j) * MID_THREADS] = acc[i][j];
    });
  }
}
