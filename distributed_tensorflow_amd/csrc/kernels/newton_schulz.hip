// Orthogonalisation of matrices by Newton-Schulz products, and the Muon update built on it.
//
//   X = G / (|G|_F + eps);   per step:  A = X X^T,  B = a I + b A + c A A,  X = B X
//
// on the orientation with m = min(rows, cols) rows of n = max(rows, cols) elements. With Muon
// around it:  V = mu V + G;  U = G + mu V (Nesterov; V without);  W = (1 - lr decay) W - lr s NS(U).
//
// Arithmetic. The three products of a step are bound by the matrix cores, and fp32 operands run
// there at a sixteenth of the 16-bit rate. So every operand is held as a pair of fp16 numbers,
// hi = fp16(x) and lo = fp16(x - hi): together 22 bits of x, at most 2^-23 of it lost (fp32 itself
// loses 2^-24). A product is hi hi + hi lo + lo hi with fp32 accumulation; lo lo (2^-22 of the
// term) is left out. Polynomial steps grow a small singular value by up to `a` each and carry the
// rounding noise of the operands along, 485-fold over five default steps: single 16-bit operands
// are off by 1e-2 of the result's size on matrices of bounded rank, this form by less than an
// fp32 computation is (its accumulators take 32 or 64 terms at a time). fp16 and not bf16
// because 11 + 11 bits in three products do what bf16 needs six for; its range is met by powers
// of two: entries of X are at most 3.5 in size (host-checked for the coefficients), stored times
// 2^14; A and B times 2^12.
//
// Work. A and B are symmetric: only tiles on and below the diagonal are computed, each written
// to both places. a I is part of B, so X is not read again for the sum. B X needs the columns of
// X where A = X X^T needs its rows: the epilogue that makes X writes it in both orders, and all
// operands are K-contiguous. The matrices of one call (up to NS_MAX_MATS, any shapes) share each
// launch: a call takes 2 + 3 steps launches whatever the count.
//
// Layout. "Split rows": row r of K elements takes 4 bytes per element, in chunks of 32 elements:
// 32 hi halves (64 bytes), then 32 lo halves. A chunk is 128 bytes, so a K-tile of 32 elements has
// the LDS image of a 64-element bf16 K-tile (16-byte pieces, XOR-swizzled by row) and lands there
// by 16-byte LDS-DMA. Rows are padded with zeros to whole chunks; edge tiles read the last row
// again instead of rows that are not there.
#include "common.h"

namespace {

constexpr int NS_MAX_MATS = 16;
constexpr int NS_MAX_STEPS = 32;
constexpr int NS_MAX_PARTS = 512;      // workgroups that share a matrix's sum of squares
constexpr float X_SCALE = 16384.f, AB_SCALE = 4096.f;
constexpr double X_LIMIT = 3.5, AB_LIMIT = 15.0;   // times the scales: below fp16's 65504

typedef __attribute__((address_space(3))) void lds_void;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

enum { NS_F32 = 0, NS_BF16 = 1, NS_F16 = 2 };
enum { TO_A = 0, TO_B = 1, TO_X = 2, TO_OUT = 3 };

struct NsMat {
  const void* g;       // [rows, cols], contiguous
  void* out;           // [rows, cols]; Muon: the weight
  float* v;            // Muon: momentum
  double* parts;       // [nparts] partial sums of squares
  char* x;             // split rows [m][kn]
  char* xt0;           // split rows [n][km]: read by even steps
  char* xt1;           //                     ... by odd ones
  char* a;             // split rows [m][km]
  char* b;
  int rows, cols;
  int m, n;
  int km, kn;          // m, n rounded up to whole chunks
  int nparts;
  float scale;         // Muon: s
};
struct NsArgs {
  NsMat t[NS_MAX_MATS];
  int first[NS_MAX_MATS + 1];    // first workgroup of each matrix in this launch
  int count;
};
struct NsMuon {
  const float* lr_dev;
  float lr, mu, decay;
  int nesterov;
};

__device__ __forceinline__ int matrix_of(const NsArgs& args, int id) {
  int i = 0;
  while (i + 1 < args.count && id >= args.first[i + 1]) ++i;
  return i;
}

__device__ __forceinline__ float ns_load(const void* p, long i, int type) {
  if (type == NS_F32) return ((const float*)p)[i];
  if (type == NS_BF16) return dtf_bf16_to_f32(((const unsigned short*)p)[i]);
  return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void ns_store(void* p, long i, int type, float v) {
  if (type == NS_F32) ((float*)p)[i] = v;
  else if (type == NS_BF16) ((unsigned short*)p)[i] = dtf_f32_to_bf16(v);
  else ((_Float16*)p)[i] = (_Float16)v;
}

// hi | lo << 16
__device__ __forceinline__ unsigned split_pack(float v) {
  const _Float16 hi = (_Float16)v;
  const _Float16 lo = (_Float16)(v - (float)hi);
  return (unsigned)__builtin_bit_cast(unsigned short, hi) |
         (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
}

// eight packed elements -> 16 bytes of hi, 16 bytes of lo
__device__ __forceinline__ void store_split8(char* chunk_hi, const unsigned* p) {
  u32x4 hi, lo;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    hi[k] = (p[2 * k] & 0xffffu) | p[2 * k + 1] << 16;
    lo[k] = p[2 * k] >> 16 | (p[2 * k + 1] & 0xffff0000u);
  }
  *reinterpret_cast<u32x4*>(chunk_hi) = hi;
  *reinterpret_cast<u32x4*>(chunk_hi + 64) = lo;
}

// byte offset of element c in a split row (its hi half; the lo half is 64 bytes further)
__device__ __forceinline__ long split_off(int c) { return (long)(c >> 5) * 128 + (c & 31) * 2; }

// ---- momentum and sum of squares -------------------------------------------------------------
// Squares are summed in 64 bits: gradients of 1e-20 or 1e+25 have squares fp32 does not hold.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs args, int type, NsMuon mo) {
  const int mat = matrix_of(args, blockIdx.x);
  const NsMat& t = args.t[mat];
  const int part = blockIdx.x - args.first[mat];
  const long total = (long)t.rows * t.cols;
  double s = 0.0;
  for (long i = part * 256L + threadIdx.x; i < total; i += t.nparts * 256L) {
    float u = ns_load(t.g, i, type);
    if (MUON) {
      const float v = __builtin_fmaf(mo.mu, t.v[i], u);
      t.v[i] = v;
      u = mo.nesterov ? __builtin_fmaf(mo.mu, v, u) : v;
    }
    s = __builtin_fma((double)u, (double)u, s);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  __shared__ double sh[4];
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) t.parts[part] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// ---- X and its transpose in split rows -------------------------------------------------------
// One 64 x 64 tile of G per workgroup: its rows go to one of the two orders as they are, its
// columns through LDS to the other.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_split_kernel(NsArgs args, int type, float eps,
                                                       NsMuon mo) {
  __shared__ unsigned tr[64 * 68];
  __shared__ double sh[4];
  const int mat = matrix_of(args, blockIdx.x);
  const NsMat& t = args.t[mat];
  const int tile = blockIdx.x - args.first[mat];
  const int tiles_c = (t.cols + 63) / 64;
  const int r0 = tile / tiles_c * 64, c0 = tile % tiles_c * 64;
  double s = 0.0;
  for (int p = threadIdx.x; p < t.nparts; p += 256) s += t.parts[p];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  // (the quotient is taken in 64 bits as well: a norm may lie beyond fp32's range)
  const double mul = (double)X_SCALE / (__builtin_sqrt(s) + (double)eps);
  const bool tall = t.rows > t.cols;
  char* direct = tall ? t.xt0 : t.x;               // rows of `cols` elements
  char* turned = tall ? t.x : t.xt0;               // rows of `rows` elements
  const long direct_pitch = 4L * (tall ? t.km : t.kn);
  const long turned_pitch = 4L * (tall ? t.kn : t.km);
  const int c8 = (threadIdx.x & 7) * 8, c = c0 + c8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rl = (threadIdx.x >> 3) + 32 * h, r = r0 + rl;
    unsigned p[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float u = 0.f;
      if (r < t.rows && c + k < t.cols) {
        const long i = (long)r * t.cols + c + k;
        u = ns_load(t.g, i, type);
        if (MUON) {
          const float v = t.v[i];                  // already advanced
          u = mo.nesterov ? __builtin_fmaf(mo.mu, v, u) : v;
        }
        u = (float)((double)u * mul);
      }
      p[k] = split_pack(u);
      tr[(c8 + k) * 68 + rl] = p[k];
    }
    // (a chunk that starts inside the row belongs to it as a whole)
    if (r < t.rows && (c & ~31) < t.cols) store_split8(direct + r * direct_pitch + split_off(c), p);
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int cl = (threadIdx.x >> 3) + 32 * h;
    if (c0 + cl < t.cols && ((r0 + c8) & ~31) < t.rows) {
      unsigned p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = tr[cl * 68 + c8 + k];
      store_split8(turned + (c0 + cl) * turned_pitch + split_off(r0 + c8), p);
    }
  }
}

// ---- the products ----------------------------------------------------------------------------
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const char* base) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0xffffffff, 0x00020000);
}

// byte offset of 16-byte piece kc of a row inside an operand tile (rows of 128 bytes)
__device__ __forceinline__ int piece_off(int row, int kc) {
  return row * 128 + ((kc ^ ((row >> 1) & 7)) << 4);
}

// One T x T tile of P Q^T, P [M][K] and Q [N][K] in split rows, by four waves of T/2 x T/2.
// Two K-tile buffers: the requests for the next K-tile are in flight while this one multiplies.
// TO_A / TO_B: symmetric results (M = N, tiles on and below the diagonal), written to both
// places; TO_X: written in both orders; TO_OUT: the caller's type.
template <int T, int TO, bool MUON>
__device__ __forceinline__ void ns_product_body(const NsArgs& args, int step, int type, float ca,
                                                float cb, float cc, const NsMuon& mo) {
  constexpr int NI = T / 32;                    // 16 x 16 tiles per wave and direction
  constexpr int WT = T / 2;
  constexpr int OP_BYTES = T * 128, BUF_BYTES = 2 * OP_BYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 1, wc = wave & 1;
  const int id = dtf_xcd_remap(blockIdx.x, gridDim.x);
  const int mat = matrix_of(args, id);
  const NsMat& t = args.t[mat];
  const int tile = id - args.first[mat];

  const bool tall = t.rows > t.cols;
  const char *P, *Q;
  int M, N, K;
  if (TO == TO_A) {
    P = Q = t.x; M = N = t.m; K = t.kn;
  } else if (TO == TO_B) {
    P = Q = t.a; M = N = t.m; K = t.km;
  } else {
    const char* xt = (step & 1) ? t.xt1 : t.xt0;
    K = t.km;
    if (TO == TO_OUT && tall) {                 // X^T = X^T B: the result as the caller lays it
      P = xt; Q = t.b; M = t.n; N = t.m;
    } else {
      P = t.b; Q = xt; M = t.m; N = t.n;
    }
  }
  int tm, tn;
  if (TO == TO_A || TO == TO_B) {
    tm = (int)((__builtin_sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= tile) ++tm;
    while (tm * (tm + 1) / 2 > tile) --tm;
    tn = tile - tm * (tm + 1) / 2;
  } else {
    constexpr int GROUP = 8;
    const int tiles_m = (M + T - 1) / T, tiles_n = (N + T - 1) / T;
    const int per_group = GROUP * tiles_n, grp = tile / per_group, first_m = grp * GROUP;
    const int gsize = tiles_m - first_m < GROUP ? tiles_m - first_m : GROUP;
    tm = first_m + tile % per_group % gsize;
    tn = tile % per_group / gsize;
  }
  const int m0 = tm * T, n0 = tn * T;
  const long pitch = 4L * K;

  unsigned voff_p[NI], voff_q[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int row = (wave * NI + j) * 8 + (lane >> 3);
    const int kc = (lane & 7) ^ ((row >> 1) & 7);
    const int rp = m0 + row < M ? row : M - 1 - m0, rq = n0 + row < N ? row : N - 1 - n0;
    voff_p[j] = (unsigned)rp * (unsigned)pitch + 16u * kc;
    voff_q[j] = (unsigned)rq * (unsigned)pitch + 16u * kc;
  }
  const __amdgpu_buffer_rsrc_t p_rsrc = rows_rsrc(P + m0 * pitch);
  const __amdgpu_buffer_rsrc_t q_rsrc = rows_rsrc(Q + n0 * pitch);
  auto request = [&](int kt, char* buf) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int piece = wave * NI + j;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(p_rsrc, (lds_void*)(buf + piece * 1024), 16,
                                               voff_p[j], kt * 128, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(q_rsrc, (lds_void*)(buf + OP_BYTES + piece * 1024),
                                               16, voff_q[j], kt * 128, 0, 0);
    }
  };

  f32x4 acc[NI][NI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int frow = lane & 15, fq = lane >> 4;
  const int nkt = K / 32;
  request(0, smem);
  for (int kt = 0; kt < nkt; ++kt) {
    // K-tile kt has landed for every wave, and every wave is done with the other buffer
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    const char* cur = smem + (kt & 1) * BUF_BYTES;
    if (kt + 1 < nkt) request(kt + 1, smem + ((kt + 1) & 1) * BUF_BYTES);
    f16x8 ph[NI], pl[NI], qh[NI], ql[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int rp = wr * WT + i * 16 + frow, rq = wc * WT + i * 16 + frow;
      ph[i] = *reinterpret_cast<const f16x8*>(cur + piece_off(rp, fq));
      pl[i] = *reinterpret_cast<const f16x8*>(cur + piece_off(rp, 4 + fq));
      qh[i] = *reinterpret_cast<const f16x8*>(cur + OP_BYTES + piece_off(rq, fq));
      ql[i] = *reinterpret_cast<const f16x8*>(cur + OP_BYTES + piece_off(rq, 4 + fq));
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        // (operands swapped: a lane's four results lie along N)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[j], ph[i], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[j], pl[i], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[j], ph[i], acc[i][j], 0, 0, 0);
      }
  }
  __syncthreads();                              // the buffers become the epilogue's scratch

  // lane: rows mb + 16 i, columns nb + 16 j + 0..3
  const int mb = m0 + wr * WT + frow, nb = n0 + wc * WT + 4 * fq;
  if (TO == TO_OUT) {
    const float lr = MUON ? (mo.lr_dev ? mo.lr_dev[0] : mo.lr) : 0.f;
    const float keep = 1.f - lr * mo.decay, take = lr * t.scale;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int m = mb + 16 * i;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = nb + 16 * j + r;
          if (n >= N) continue;
          const long at = (long)m * N + n;
          const float v = acc[i][j][r] * (1.f / (X_SCALE * AB_SCALE));
          if (MUON) {
            float* w = (float*)t.out;
            w[at] = __builtin_fmaf(-take, v, keep * w[at]);
          } else {
            ns_store(t.out, at, type, v);
          }
        }
    }
    return;
  }

  // packed (hi | lo << 16) results; zero behind the last row and column
  unsigned pk[NI][NI][4];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int m = mb + 16 * i, n = nb + 16 * j;
      f32x4 v = acc[i][j];
      if (TO == TO_A) v *= AB_SCALE / (X_SCALE * X_SCALE);
      if (TO == TO_X) v *= 1.f / AB_SCALE;
      if (TO == TO_B) {
        f16x4 ah = {0, 0, 0, 0}, al = {0, 0, 0, 0};
        if (m < M && (n & ~31) < N) {
          const char* src = t.a + m * pitch + split_off(n);
          ah = *reinterpret_cast<const f16x4*>(src);
          al = *reinterpret_cast<const f16x4*>(src + 64);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = __builtin_fmaf(cc / AB_SCALE, v[r],
                                __builtin_fmaf(cb, (float)ah[r] + (float)al[r],
                                               m == n + r ? ca * AB_SCALE : 0.f));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        pk[i][j][r] = m < M && n + r < N ? split_pack(v[r]) : 0u;
    }

  char* D = TO == TO_A ? t.a : TO == TO_B ? t.b : t.x;          // rows along M
  char* E = TO == TO_X ? ((step & 1) ? t.xt0 : t.xt1) : D;      // rows along N
  const long d_pitch = 4L * (TO == TO_X ? t.kn : t.km), e_pitch = 4L * t.km;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int m = mb + 16 * i, n = nb + 16 * j;
      if (m < M && (n & ~31) < N) {
        char* dst = D + m * d_pitch + split_off(n);
        const unsigned* p = pk[i][j];
        *reinterpret_cast<uint2*>(dst) = uint2{(p[0] & 0xffffu) | p[1] << 16,
                                               (p[2] & 0xffffu) | p[3] << 16};
        *reinterpret_cast<uint2*>(dst + 64) = uint2{p[0] >> 16 | (p[1] & 0xffff0000u),
                                                    p[2] >> 16 | (p[3] & 0xffff0000u)};
      }
    }
  if ((TO == TO_A || TO == TO_B) && tm == tn) return;   // a diagonal tile is its own mirror image
  // the other order through a strip of LDS per wave: [WT of N][32 of M], rows of 36 dwords
  unsigned* strip = reinterpret_cast<unsigned*>(smem) + wave * (WT * 36);
#pragma unroll
  for (int h = 0; h < NI / 2; ++h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          strip[(16 * j + 4 * fq + r) * 36 + 16 * i + frow] = pk[2 * h + i][j][r];
    __builtin_amdgcn_wave_barrier();
    const int mc = m0 + wr * WT + 32 * h;               // first element of the chunk
#pragma unroll
    for (int q = 0; q < NI; ++q) {
      const int nl = 16 * q + (lane >> 2), n = n0 + wc * WT + nl;
      unsigned p[8];
      const u32x4* src = reinterpret_cast<const u32x4*>(strip + nl * 36 + (lane & 3) * 8);
      *reinterpret_cast<u32x4*>(p) = src[0];
      *reinterpret_cast<u32x4*>(p + 4) = src[1];
      if (n < N && mc < M) store_split8(E + n * e_pitch + split_off(mc + (lane & 3) * 8), p);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int T, int TO, bool MUON>
__global__ __launch_bounds__(256) void ns_product_kernel(NsArgs args, int step, int type,
                                                         float ca, float cb, float cc, NsMuon mo) {
  ns_product_body<T, TO, MUON>(args, step, type, ca, cb, cc, mo);
}

// ---- host ------------------------------------------------------------------------------------
long up(long v, long to) { return (v + to - 1) / to * to; }

struct NsSizes {
  long m, n, km, kn, parts;
  long x, xt, sq;                 // bytes of one image
  long total;
};
NsSizes sizes_of(long rows, long cols) {
  NsSizes s;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  s.km = up(s.m, 32);
  s.kn = up(s.n, 32);
  const long want = (rows * cols + 4095) / 4096;
  s.parts = want < NS_MAX_PARTS ? want : NS_MAX_PARTS;
  s.x = up(4 * s.m * s.kn, 256);
  s.xt = up(4 * s.n * s.km, 256);
  s.sq = up(4 * s.m * s.km, 256);
  s.total = up(8 * s.parts, 256) + s.x + 2 * s.xt + 2 * s.sq;
  return s;
}

bool bad_shape(long rows, long cols) {
  return rows < 1 || cols < 1 || rows > (1L << 22) || cols > (1L << 22);
}

// Sizes of X, A and B over the steps, from the singular values' side: s in [0, r] -> p(s). The
// stored fp16 images must hold every entry, and an entry is at most the largest singular value.
bool coefficients_fit(int steps, const float* coef) {
  double r = 1.0 + 1e-6;
  for (int k = 0; k < steps; ++k) {
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
    double top = 0.0, b_top = 0.0;
    constexpr int GRID = 4096;
    for (int i = 0; i <= GRID; ++i) {
      const double s = r * i / GRID, t = s * s;
      const double q = a + b * t + c * t * t;
      if (!(q == q)) return false;
      b_top = fmax(b_top, fabs(q));
      top = fmax(top, fabs(s * q));
    }
    if (!(r * r <= AB_LIMIT) || !(b_top <= AB_LIMIT) || !(top <= X_LIMIT)) return false;
    r = top * (1.0 + 1e-3);              // between grid points, and for rounding
  }
  return true;
}

template <typename KernelT>
void allow_lds(KernelT kernel, int lds) {
  (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <int T, bool MUON>
int launch_steps(NsArgs& args, int type, int steps, const float* coef, const NsMuon& mo,
                 hipStream_t stream) {
  constexpr int LDS = 2 * 2 * T * 128;
  static_assert(4 * (T / 2) * 36 * 4 <= LDS, "the epilogue's strips fit the K-tile buffers");
  static DtfPerDeviceOnce once;
  dtf_once_per_device(once, [&] {
    allow_lds(ns_product_kernel<T, TO_A, false>, LDS);
    allow_lds(ns_product_kernel<T, TO_B, false>, LDS);
    allow_lds(ns_product_kernel<T, TO_X, false>, LDS);
    allow_lds(ns_product_kernel<T, TO_OUT, MUON>, LDS);
  });
  NsArgs sym = args, full = args;
  for (int i = 0; i < args.count; ++i) {
    const int tm = (args.t[i].m + T - 1) / T, tn = (args.t[i].n + T - 1) / T;
    sym.first[i + 1] = sym.first[i] + tm * (tm + 1) / 2;
    full.first[i + 1] = full.first[i] + tm * tn;
  }
  const dim3 gs(sym.first[args.count]), gf(full.first[args.count]), block(256);
  for (int k = 0; k < steps; ++k) {
    const float a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
    hipLaunchKernelGGL((ns_product_kernel<T, TO_A, false>), gs, block, LDS, stream, sym, k, type,
                       a, b, c, mo);
    hipLaunchKernelGGL((ns_product_kernel<T, TO_B, false>), gs, block, LDS, stream, sym, k, type,
                       a, b, c, mo);
    if (k + 1 < steps)
      hipLaunchKernelGGL((ns_product_kernel<T, TO_X, false>), gf, block, LDS, stream, full, k,
                         type, a, b, c, mo);
    else
      hipLaunchKernelGGL((ns_product_kernel<T, TO_OUT, MUON>), gf, block, LDS, stream, full, k,
                         type, a, b, c, mo);
  }
  DTF_LAUNCH_CHECK();
  return DTF_OK;
}

template <bool MUON>
int run(int count, const void* const* g, void* const* out, float* const* v, const float* scale,
        const int* rows, const int* cols, int type, int steps, const float* coef, float eps,
        const NsMuon& mo, void* workspace, long workspace_bytes, hipStream_t stream) {
  if (count < 0 || count > NS_MAX_MATS || type < NS_F32 || type > NS_F16 || steps < 1 ||
      steps > NS_MAX_STEPS || !coef || !(eps >= 0.f) ||
      (count > 0 && (!g || !out || !rows || !cols || !workspace)))
    return DTF_ERR_BAD_ARG;
  if (count == 0) return DTF_OK;
  if (!coefficients_fit(steps, coef)) return DTF_ERR_UNSUPPORTED;
  NsArgs args = {};
  args.count = count;
  char* at = (char*)workspace;
  long used = 0, tiles128 = 0;
  if ((uintptr_t)at & 255) return DTF_ERR_BAD_ARG;
  NsArgs parts, split;
  for (int i = 0; i < count; ++i) {
    if (bad_shape(rows[i], cols[i]) || !g[i] || !out[i] || (MUON && (!v[i])))
      return DTF_ERR_BAD_ARG;
    const NsSizes s = sizes_of(rows[i], cols[i]);
    NsMat& t = args.t[i];
    t.g = g[i];
    t.out = out[i];
    t.v = MUON ? v[i] : nullptr;
    t.scale = MUON ? scale[i] : 1.f;
    t.rows = rows[i];
    t.cols = cols[i];
    t.m = (int)s.m;
    t.n = (int)s.n;
    t.km = (int)s.km;
    t.kn = (int)s.kn;
    t.nparts = (int)s.parts;
    used += s.total;
    if (used > workspace_bytes) return DTF_ERR_BAD_ARG;
    t.parts = (double*)at;
    at += up(8 * s.parts, 256);
    t.x = at;
    at += s.x;
    t.xt0 = at;
    at += s.xt;
    t.xt1 = at;
    at += s.xt;
    t.a = at;
    at += s.sq;
    t.b = at;
    at += s.sq;
    tiles128 += ((s.m + 127) / 128) * ((s.n + 127) / 128);
  }
  parts = split = args;
  for (int i = 0; i < count; ++i) {
    const long tiles = ((rows[i] + 63L) / 64) * ((cols[i] + 63L) / 64);
    if (split.first[i] + tiles > (1L << 30)) return DTF_ERR_UNSUPPORTED;
    parts.first[i + 1] = parts.first[i] + args.t[i].nparts;
    split.first[i + 1] = split.first[i] + (int)tiles;
  }
  hipLaunchKernelGGL((ns_norm_kernel<MUON>), dim3(parts.first[count]), dim3(256), 0, stream, parts,
                     type, mo);
  hipLaunchKernelGGL((ns_split_kernel<MUON>), dim3(split.first[count]), dim3(256), 0, stream,
                     split, type, eps, mo);
  DTF_LAUNCH_CHECK();
  // 128 x 128 tiles once they give the chip's 256 CUs two workgroups each
  return tiles128 >= 512 ? launch_steps<128, MUON>(args, type, steps, coef, mo, stream)
                         : launch_steps<64, MUON>(args, type, steps, coef, mo, stream);
}

}  // namespace

// bytes of workspace (256-byte aligned) for `count` matrices; 0 for shapes that are not taken
DTF_API long dtf_newton_schulz_workspace(int count, const int* rows, const int* cols) {
  if (count < 0 || count > NS_MAX_MATS || (count > 0 && (!rows || !cols))) return 0;
  long total = 256;
  for (int i = 0; i < count; ++i) {
    if (bad_shape(rows[i], cols[i])) return 0;
    total += sizes_of(rows[i], cols[i]).total;
  }
  return total;
}

// out[i] = orthogonalised g[i], both [rows[i], cols[i]] contiguous of `type` (0 fp32, 1 bf16,
// 2 fp16), for up to 16 matrices in one sequence of launches. coef: (a, b, c) of every step;
// coefficients under which a singular value in [0, 1] grows beyond 3.5 are refused
// (DTF_ERR_UNSUPPORTED).
DTF_API int dtf_newton_schulz(int count, const void* const* g, void* const* out, const int* rows,
                              const int* cols, int type, int steps, const float* coef, float eps,
                              void* workspace, long workspace_bytes, hipStream_t stream) {
  return run<false>(count, g, out, nullptr, nullptr, rows, cols, type, steps, coef, eps, NsMuon{},
                    workspace, workspace_bytes, stream);
}

// The Muon update of up to 16 fp32 weights w[i] [rows[i], cols[i]] and their momenta v[i] from
// g[i], in place. scale[i] multiplies the learning rate; lr_dev: device scalar that replaces lr.
DTF_API int dtf_multi_muon_f32(int count, float* const* w, const float* const* g, float* const* v,
                               const float* scale, const int* rows, const int* cols, int steps,
                               const float* coef, float eps, float lr, const float* lr_dev,
                               float mu, int nesterov, float decay, void* workspace,
                               long workspace_bytes, hipStream_t stream) {
  if (count > 0 && (!v || !scale)) return DTF_ERR_BAD_ARG;
  NsMuon mo = {lr_dev, lr, mu, decay, nesterov};
  return run<true>(count, (const void* const*)g, (void* const*)w, v, scale, rows, cols, NS_F32,
                   steps, coef, eps, mo, workspace, workspace_bytes, stream);
}
