// Orthogonalisation of matrices by Newton-Schulz products, and the Muon update built on it.
//
//   X = G / (|G|_F + eps);   per step:  A = X X^T,  B = a I + b A + c A A,  X = B X
//
// on the orientation with m = min(rows, cols) rows of n = max(rows, cols) elements. With Muon
// around it:  V = mu V + G;  U = G + mu V (Nesterov; V without);  W = (1 - lr decay) W - lr s NS(U).
//
// Arithmetic. The three products of a step are bound by the matrix cores, and fp32 operands run
// there at a sixteenth of the 16-bit rate. So every operand is held as a pair of fp16 numbers,
// hi = fp16(x) and lo = fp16(2^11 (x - hi)): together 22 bits of x, at most 2^-23 of it lost (fp32
// itself loses 2^-24). A product is hi hi + 2^-11 (hi lo + lo hi) with fp32 accumulation, the two
// parts in accumulators of their own; lo lo (2^-22 of the term) is left out. fp16 and not bf16
// because 11 + 11 bits in three products do what bf16 needs six for; its range is met by powers
// of two: entries of X are at most 3.5 in size (host-checked for the coefficients), stored times
// 2^14; A and B times 2^12. The factor 2^11 of lo keeps both halves normal numbers for entries of
// X down to 2^-28 and of A and B down to 2^-26; below, an entry is off by at most 2^-50 and 2^-48.
// So a row that is eight decades smaller than the others keeps its own digits, as it does in
// fp32: 4096 x 8192 with rows spread over eight decades, the worst row is off by 5e-5 of itself
// (fp32 4e-5; with lo = x - hi unscaled 1e-1). The factor costs up to 1 % of the time.
//
// Polynomial steps grow a small singular value by up to `a` each and carry the rounding noise of
// the operands along, 485-fold over five default steps: single 16-bit operands are off by 1e-2 of
// the result's size on matrices of bounded rank, this form by less than an fp32 computation is
// (its sums hold 128 elements before they are emptied).
//
// Work. A and B are symmetric: only tiles on and below the diagonal are computed, each written
// to both places. a I is part of B, so X is not read again for the sum. B X needs the columns of
// X where A = X X^T needs its rows: the epilogue that makes X writes it in both orders, and all
// operands are K-contiguous. Long matrices take two steps as one (step_pairs), which leaves out
// every other pair of products with X. The matrices of one call (up to NS_MAX_MATS, any shapes)
// share each launch: two, and three per step, whatever the count; long ones may have a sequence of
// their own, and matrices of up to 64 rows or columns have (newton_schulz_thin.h). Calls of nothing
// larger than 128 x 2048 take one or two steps in a launch (newton_schulz_mid.h).
//
// Layout. An image of a matrix is a row of K-tiles of 32 columns; in a K-tile every row has 128
// bytes: 32 hi halves, then 32 lo halves. So the rows of a K-tile that a workgroup wants lie in one
// piece (with whole rows one behind the other, 4 K bytes apart, 1500 x 1500 took 408 us instead of
// 391, 8192 x 4096 5.42 ms instead of 5.39), have the LDS image of a 64-element bf16 K-tile (16-byte
// pieces, XOR-swizzled by row) and land there by 16-byte LDS-DMA. Columns are padded with zeros to
// whole K-tiles; edge tiles read the last row again instead of rows that are not there.
#include "elem.h"

namespace {

constexpr int NS_CHAIN = 4;            // K-tiles an accumulator runs through before it is emptied
constexpr int NS_MAX_MATS = 16;
constexpr int NS_MAX_STEPS = 32;
constexpr int NS_SLOTS = 512;          // workgroups of a product that run at once, at most
constexpr int NS_MAX_PARTS = 1024;     // workgroups that share a matrix's sum of squares
constexpr float X_SCALE = 16384.f, AB_SCALE = 4096.f;
constexpr float LO_SCALE = 2048.f;     // of the small halves
constexpr double X_LIMIT = 3.5, AB_LIMIT = 15.0;   // times the scales: below fp16's 65504

typedef __attribute__((address_space(3))) void lds_void;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct yes {
  static constexpr int value = 1;
};
struct no {
  static constexpr int value = 0;
};

enum { NS_F32 = 0, NS_BF16 = 1, NS_F16 = 2 };
enum { TO_A = 0, TO_B = 1, TO_S = 2, TO_X = 3, TO_OUT = 4 };

struct NsMat {
  const void* g;       // [rows, cols], contiguous
  void* out;           // [rows, cols]; Muon: the weight
  float* v;            // Muon: momentum
  double* parts;       // [nparts] partial sums of squares
  char* x;             // image of [m][kn]
  char* xt0;           // image of [n][km]: read by even steps
  char* xt1;           //                     ... by odd ones
  char* sq[3];         // image of [m][km]: A, B and products of them
  int rows, cols;
  int m, n;
  int km, kn;          // m, n rounded up to whole K-tiles
  int nparts;
  float scale;         // Muon: s
  double* gram;        // thin matrices: [slabs][lower 16 x 16 tiles][256]
  int slabs, slab_cols;
  char* a_parts[2];    // up to 128 x 2048: the slabs' parts of A, read and written in turn
};
struct NsArgs {
  NsMat t[NS_MAX_MATS];
  int first[NS_MAX_MATS + 1];    // first tile (or workgroup) of each matrix in this launch
  int count;
  // products: tiles [0, unsplit) have a workgroup each; every later tile has `splits`
  // workgroups that share its K range
  int unsplit, splits;
  int p, q, to;                  // which of sq: first and second operand, result
  float* partial;                // [(tile - unsplit) * splits + split][T * T]
  int* arrived;                  // [tile - unsplit], zero between launches
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

// hi | lo << 16
__device__ __forceinline__ unsigned split_pack(float v) {
  const _Float16 hi = (_Float16)v;
  const _Float16 lo = (_Float16)((v - (float)hi) * LO_SCALE);
  return (unsigned)__builtin_bit_cast(unsigned short, hi) |
         (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
}

// four elements' hi halves and lo halves (two conversions in an instruction)
__device__ __forceinline__ void split4(f32x4 v, uint2& hi, uint2& lo) {
  const f16x2 h0 = __builtin_convertvector(f32x2{v[0], v[1]}, f16x2);
  const f16x2 h1 = __builtin_convertvector(f32x2{v[2], v[3]}, f16x2);
  const f32x2 r0 = {(v[0] - (float)h0[0]) * LO_SCALE, (v[1] - (float)h0[1]) * LO_SCALE};
  const f32x2 r1 = {(v[2] - (float)h1[0]) * LO_SCALE, (v[3] - (float)h1[1]) * LO_SCALE};
  hi = uint2{__builtin_bit_cast(unsigned, h0), __builtin_bit_cast(unsigned, h1)};
  lo = uint2{__builtin_bit_cast(unsigned, __builtin_convertvector(r0, f16x2)),
             __builtin_bit_cast(unsigned, __builtin_convertvector(r1, f16x2))};
}

__device__ __forceinline__ float joined(_Float16 hi, _Float16 lo) {
  return __builtin_fmaf((float)lo, 1.f / LO_SCALE, (float)hi);
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

// byte offset of element c of row r in an image of `rows` rows (its hi half; the lo half is 64
// bytes further)
__device__ __forceinline__ long image_off(int rows, int r, int c) {
  return ((long)(c >> 5) * rows + r) * 128 + (c & 31) * 2;
}

// ---- momentum and sum of squares -------------------------------------------------------------
// Squares are summed in 64 bits: gradients of 1e-20 or 1e+25 have squares fp32 does not hold.
template <typename E, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs args, NsMuon mo) {
  constexpr int V = 16 / (int)sizeof(E);
  const int mat = matrix_of(args, blockIdx.x);
  const NsMat& t = args.t[mat];
  const int part = blockIdx.x - args.first[mat];
  const long total = (long)t.rows * t.cols, stride = t.nparts * 256L * V;
  const E* g = (const E*)t.g;
  double s = 0.0;
#pragma unroll 4
  for (long i = (part * 256L + threadIdx.x) * V; i < total; i += stride) {
    const int n = total - i < V ? (int)(total - i) : V;
    float u[V];
    load_part<V>(g + i, 0, n, u);
    if (MUON) {
      float v[V];
      load_part<V>(t.v + i, 0, n, v);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[k] = __builtin_fmaf(mo.mu, v[k], u[k]);
        u[k] = mo.nesterov ? __builtin_fmaf(mo.mu, v[k], u[k]) : v[k];
      }
      store_part<V>(t.v + i, 0, n, v);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s = __builtin_fma((double)u[k], (double)u[k], s);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  __shared__ double sh[4];
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) t.parts[part] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < NS_SLOTS; i += 256) args.arrived[i] = 0;
}

// ---- X and its transpose as images -----------------------------------------------------------
// One 64 x 64 tile of G per workgroup: its rows go to one of the two orders as they are, its
// columns through LDS to the other.
template <typename E, bool MUON>
__global__ __launch_bounds__(256) void ns_split_kernel(NsArgs args, float eps, NsMuon mo) {
  // (rows of 65 dwords: the 8 x 8 lanes of a wave meet 64 banks both ways)
  __shared__ unsigned tr[64 * 65];
  __shared__ double sh[4];
  const int mat = matrix_of(args, blockIdx.x);
  const NsMat& t = args.t[mat];
  const int tile = blockIdx.x - args.first[mat];
  const int tiles_c = (t.cols + 63) / 64;
  const int r0 = tile / tiles_c * 64, c0 = tile % tiles_c * 64;
  const int c8 = (threadIdx.x & 7) * 8, c = c0 + c8;
  float u[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + (threadIdx.x >> 3) + 32 * h;
    const int n = r < t.rows ? t.cols : 0;
    const long at = (long)(r < t.rows ? r : 0) * t.cols;
    load_part<8>((const E*)t.g + at, c, n, u[h]);
    if (MUON) {
      float v[8];                                  // already advanced
      load_part<8>(t.v + at, c, n, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[h][k] = mo.nesterov ? __builtin_fmaf(mo.mu, v[k], u[h][k]) : v[k];
    }
  }
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
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rl = (threadIdx.x >> 3) + 32 * h, r = r0 + rl;
    unsigned p[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // (0 / 0 of a zero matrix without epsilon stays in the matrix: padding is zero always)
      p[k] = r < t.rows && c + k < t.cols ? split_pack((float)((double)u[h][k] * mul)) : 0u;
      tr[(c8 + k) * 65 + rl] = p[k];
    }
    // (a chunk that starts inside the row belongs to it as a whole)
    if (r < t.rows && (c & ~31) < t.cols) store_split8(direct + image_off(t.rows, r, c), p);
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int cl = (threadIdx.x >> 3) + 32 * h;
    if (c0 + cl < t.cols && ((r0 + c8) & ~31) < t.rows) {
      unsigned p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = tr[cl * 65 + c8 + k];
      store_split8(turned + image_off(t.cols, c0 + cl, r0 + c8), p);
    }
  }
}

// ---- the products ----------------------------------------------------------------------------
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const char* base) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0xffffffff, 0x00020000);
}

// rows r0 and on of K-tile kt
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const char* image, int rows, int r0,
                                                            int kt) {
  return rows_rsrc(image + ((long)kt * rows + r0) * 128);
}

// Workgroups that share a K range of kt K-tiles when `most` are offered. Parts go through memory
// and are waited for, 8 us a product at 1024 x 1024: a split is made where it takes 40 K-tiles or
// more (0.2 us each on 64 x 64 tiles) out of a workgroup's way, in parts of 16 or more. Whole
// call, split as here / never / as often as offered: 1024 x 1024 183 / 182 / 247 us, 2048 x 2048
// 714 / 766 / 716, 300 x 8000 175 / 275 / 174, 1024 x 4096 316 / 327 / 355, 1024 x 8192 421 / 458 /
// 458, 8192 x 4096 5.33 / 7.52 / 5.31 ms.
__host__ __device__ __forceinline__ int split_count(int kt, int most) {
  int s = kt / 16;
  s = s < most ? s : most;
  return s > 1 && kt - kt / s >= 40 ? s : 1;
}

// byte offset of 16-byte piece kc of a row inside an operand tile (rows of 128 bytes)
__device__ __forceinline__ int piece_off(int row, int kc) {
  return row * 128 + ((kc ^ ((row >> 1) & 7)) << 4);
}

// One BM x BN tile of P Q^T, images of P [M][K] and Q [N][K]. TO_A (X X^T), TO_B (a I + b A +
// c A A) and TO_S (a product of polynomials of one A): symmetric results (M = N, tiles on and
// below the diagonal), written to both places; TO_X: written in both orders; TO_OUT: the caller's
// type.
//
// Accumulation. The matrix instruction adds its 32 products to the accumulator in steps of its
// own; a long chain of them loses what the pairs gain (a gradient of 1024 x 1024: the result was off
// by 3.0e-6, an fp32 computation by 3.1e-6). Every NS_CHAIN K-tiles the accumulators of hi hi are
// added to a second set and start again from zero (1.8e-6; no time). The products with the small
// halves count 2^-11 of themselves and stay in one chain.
//
// Splits. A tile whose K range is shared leaves fp32 partial tiles in memory; the workgroup that
// arrives last adds all of them in split order, whoever it is, so the bits do not depend on the
// order of arrival.
struct NsTile {
  const char *P, *Q;
  int M, N, K;
  int m0, n0;
  int kt0, nkt;              // this workgroup's K-tiles
  int mat, shared, split, splits;
};

template <int NM, int NN>
__device__ __forceinline__ void add_cross(f32x4 (&sum)[NM][NN], const f32x4 (&cross)[NM][NN]) {
#pragma unroll
  for (int i = 0; i < NM; ++i)
#pragma unroll
    for (int j = 0; j < NN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sum[i][j][r] = __builtin_fmaf(cross[i][j][r], 1.f / LO_SCALE, sum[i][j][r]);
}

// this workgroup's tile; false: nothing to do
template <int BM, int BN, int TO>
__device__ __forceinline__ bool ns_locate(const NsArgs& args, int step, NsTile& w) {
  int id;
  w.split = 0;
  w.splits = 1;
  if ((int)blockIdx.x < args.unsplit) {
    id = dtf_xcd_remap(blockIdx.x, args.unsplit);
  } else {
    // an XCD takes neighbouring tiles of one K range, whose rows its L2 holds (the parts of a tile
    // side by side instead, so on several XCDs: 1024 x 8192 in single steps 726 us, here 617)
    const int rest = args.first[args.count] - args.unsplit;
    w.splits = args.splits;
    const int r = dtf_xcd_remap(blockIdx.x - args.unsplit, rest * w.splits);
    id = args.unsplit + r % rest;
    w.split = r / rest;
  }
  w.shared = id - args.unsplit;
  w.mat = matrix_of(args, id);
  const NsMat& t = args.t[w.mat];
  const int tile = id - args.first[w.mat];
  if (TO == TO_A) {
    w.P = w.Q = t.x; w.M = w.N = t.m; w.K = t.kn;
  } else if (TO == TO_B || TO == TO_S) {
    w.P = t.sq[args.p]; w.Q = t.sq[args.q]; w.M = w.N = t.m; w.K = t.km;
  } else {
    const char* xt = (step & 1) ? t.xt1 : t.xt0;
    w.K = t.km;
    if (TO == TO_OUT && t.rows > t.cols) {      // X^T = X^T B: the result as the caller lays it
      w.P = xt; w.Q = t.sq[args.p]; w.M = t.n; w.N = t.m;
    } else {
      w.P = t.sq[args.p]; w.Q = xt; w.M = t.m; w.N = t.n;
    }
  }
  const int all_kt = w.K / 32;
  if (w.splits > 1) {                           // (a matrix with a short K uses fewer)
    w.splits = split_count(all_kt, w.splits);
    if (w.split >= w.splits) return false;
  }
  w.kt0 = (int)((long)all_kt * w.split / w.splits);
  w.nkt = (int)((long)all_kt * (w.split + 1) / w.splits) - w.kt0;
  int tm, tn;
  if (TO == TO_A || TO == TO_B || TO == TO_S) {
    // row tm of the triangle has F (tm + 1) tiles: F tm (tm + 1) / 2 before it
    constexpr int F = BM / BN;
    tm = (int)((__builtin_sqrtf(8.f / F * tile + 1.f) - 1.f) * 0.5f);
    while (F * (tm + 1) * (tm + 2) / 2 <= tile) ++tm;
    while (F * tm * (tm + 1) / 2 > tile) --tm;
    tn = tile - F * tm * (tm + 1) / 2;
  } else {
    constexpr int GROUP = 8;
    const int tiles_m = (w.M + BM - 1) / BM, tiles_n = (w.N + BN - 1) / BN;
    const int per_group = GROUP * tiles_n, grp = tile / per_group, first_m = grp * GROUP;
    const int gsize = tiles_m - first_m < GROUP ? tiles_m - first_m : GROUP;
    tm = first_m + tile % per_group % gsize;
    tn = tile % per_group / gsize;
  }
  w.m0 = tm * BM;
  w.n0 = tn * BN;
  return true;
}

// The parts of a shared tile. True in the workgroup that has all of them in `sum`. The XCDs' L2s
// do not see each other's lines, so the parts go through memory: stores and loads of device scope
// (sc1) pass the L2 by, and a store is complete once it has arrived there. (A release fence instead
// writes the whole L2 back, 0.4 us each and one after the other on an XCD: 29 us for a product at
// 1024 x 1024 split three ways.) The first THREADS threads hold the tile. A load from there takes
// a microsecond and more, so 8 of a thread's are on their way at once, and as many again are asked
// for before the first are added.
constexpr int SC1 = 16;
template <int NM, int NN, int THREADS>
__device__ __forceinline__ bool ns_join(f32x4 (&sum)[NM][NN], const NsArgs& args, const NsTile& w) {
  __shared__ int last;
  constexpr int FR = NM * NN, PART = FR * THREADS * 16;      // fragments and bytes of a part
  constexpr int U = 16 / FR;                                 // parts in two requests of 8 loads
  const bool holds = threadIdx.x < THREADS;
  const __amdgpu_buffer_rsrc_t parts =
      rows_rsrc((const char*)args.partial + (long)w.shared * args.splits * PART);
  const int at = threadIdx.x * 16;
  if (holds) {
#pragma unroll
    for (int f = 0; f < FR; ++f)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum[f / NN][f % NN]),
                                                 parts, at, w.split * PART + f * THREADS * 16, SC1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's part has arrived ...
  __syncthreads();                                   // ... and every wave's, before the count
  if (threadIdx.x == 0) {
    const int before = __hip_atomic_fetch_add(&args.arrived[w.shared], 1, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT);
    last = before == w.splits - 1;
    if (last)                                   // nobody else comes: ready for the next launch
      __hip_atomic_store(&args.arrived[w.shared], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last || !holds) return false;
  u32x4 v[2][8];
  // half h of the loads of parts k .. k + U - 1 (behind the last part the last one again, not added)
  auto ask = [&](int k, int h) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int part = k + (h * 8 + x) / FR, f = (h * 8 + x) % FR;
      v[h][x] = __builtin_amdgcn_raw_buffer_load_b128(
          parts, at, (part < w.splits ? part : w.splits - 1) * PART + f * THREADS * 16, SC1);
    }
  };
  auto add = [&](int k, int h) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int f = (h * 8 + x) % FR;
      if (k + (h * 8 + x) / FR < w.splits) sum[f / NN][f % NN] += __builtin_bit_cast(f32x4, v[h][x]);
    }
  };
#pragma unroll
  for (int f = 0; f < FR; ++f) sum[f / NN][f % NN] = f32x4{0.f, 0.f, 0.f, 0.f};
  ask(0, 0);
  for (int k = 0; k < w.splits; k += U) {
    ask(k, 1);
    add(k, 0);
    if (k + U < w.splits) ask(k + U, 0);
    add(k, 1);
  }
  return true;
}

// Results of one wave: rows mw + 16 i + lane % 16, columns nw + 16 j + 4 (lane / 16) + 0..3.
// `strip`: 16 NN rows of 36 dwords of LDS, this wave's own.
template <typename E, int NM, int NN, int TO, bool MUON>
__device__ __forceinline__ void ns_store(const f32x4 (&acc)[NM][NN], const NsArgs& args,
                                         const NsTile& w, int step, float ca, float cb, float cc,
                                         const NsMuon& mo, int mw, int nw, unsigned* strip) {
  const NsMat& t = args.t[w.mat];
  const int lane = threadIdx.x & 63, frow = lane & 15, fq = lane >> 4;
  const int mb = mw + frow, nb = nw + 4 * fq, M = w.M, N = w.N;
  if (TO == TO_OUT) {
    const float lr = MUON ? (mo.lr_dev ? mo.lr_dev[0] : mo.lr) : 0.f;
    const float keep = 1.f - lr * mo.decay, take = lr * t.scale;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const int m = mb + 16 * i;
      if (m >= M) continue;
      E* row = (E*)t.out + (long)m * N;
#pragma unroll
      for (int j = 0; j < NN; ++j) {
        const int n = nb + 16 * j;
        if (n >= N) continue;
        float v[4], old[4];
        if (MUON) load_part<4>(row, n, N, old);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = acc[i][j][r] * (1.f / (X_SCALE * AB_SCALE));
          if (MUON) v[r] = __builtin_fmaf(-take, v[r], keep * old[r]);
        }
        store_part<4>(row, n, N, v);
      }
    }
    return;
  }
  constexpr bool SYM = TO == TO_A || TO == TO_B || TO == TO_S;
  // (squares of this wave's size: above the diagonal the mirror image writes)
  const int row_block = mw / (16 * NM), col_block = nw / (16 * NN);
  if (SYM && row_block < col_block) return;
  char* direct = SYM ? t.sq[args.to] : t.x;                            // rows along M
  char* turned = TO == TO_X ? ((step & 1) ? t.xt0 : t.xt1) : direct;   // rows along N
#pragma unroll
  for (int h = 0; h < NM / 2; ++h) {
    // packed (hi | lo << 16) results; zero behind the last row and column
    unsigned pk[2][NN][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NN; ++j) {
        const int m = mb + 16 * (2 * h + i), n = nb + 16 * j;
        f32x4 v = acc[2 * h + i][j];
        if (TO == TO_A) v *= AB_SCALE / (X_SCALE * X_SCALE);
        if (TO == TO_X || TO == TO_S) v *= 1.f / AB_SCALE;
        if (TO == TO_B) {
          // (any address inside for the elements that are not there: they become zeros below)
          const char* src = t.sq[args.p] + image_off(M, m < M ? m : 0, (n & ~31) < N ? n : 0);
          const f16x4 ah = *reinterpret_cast<const f16x4*>(src);
          const f16x4 al = *reinterpret_cast<const f16x4*>(src + 64);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            v[r] = __builtin_fmaf(cc / AB_SCALE, v[r],
                                  __builtin_fmaf(cb, joined(ah[r], al[r]),
                                                 m == n + r ? ca * AB_SCALE : 0.f));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = m < M && n + r < N ? v[r] : 0.f;
        uint2 hi, lo;
        split4(v, hi, lo);
        unsigned* p = pk[i][j];
        p[0] = (hi.x & 0xffffu) | lo.x << 16;
        p[1] = hi.x >> 16 | (lo.x & 0xffff0000u);
        p[2] = (hi.y & 0xffffu) | lo.y << 16;
        p[3] = hi.y >> 16 | (lo.y & 0xffff0000u);
        if (m < M && (n & ~31) < N) {
          char* dst = direct + image_off(M, m, n);
          *reinterpret_cast<uint2*>(dst) = hi;
          *reinterpret_cast<uint2*>(dst + 64) = lo;
        }
      }
    if (SYM && row_block == col_block) continue;   // a diagonal block is its own mirror image
    // the other order through the strip: [16 NN of N][32 of M]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          strip[(16 * j + 4 * fq + r) * 36 + 16 * i + frow] = pk[i][j][r];
    __builtin_amdgcn_wave_barrier();
    const int mc = mw + 32 * h;                    // first element of the chunk
#pragma unroll
    for (int q = 0; q < NN; ++q) {
      const int nl = 16 * q + (lane >> 2), n = nw + nl;
      unsigned p[8];
      const u32x4* src = reinterpret_cast<const u32x4*>(strip + nl * 36 + (lane & 3) * 8);
      *reinterpret_cast<u32x4*>(p) = src[0];
      *reinterpret_cast<u32x4*>(p + 4) = src[1];
      if (n < N && mc < M) store_split8(turned + image_off(N, n, mc + (lane & 3) * 8), p);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// 64 x 64 tiles: four multiplying waves and four that issue the LDS-DMA requests, three K-tiles
// ahead into four buffers -- the multiplying waves never wait at the address unit. Two workgroups
// per CU. (Four waves that do both: 1024 x 1024 302 us instead of 186.) A workgroup that has its CU to
// itself takes 0.23 us per K-tile: every 16 KB has a wait and a barrier of its own, and their
// latency is what bounds it. (LDS-DMA alone brings 16 KB in 0.07 us, with a barrier per 64 KB in
// 0.12, profiles/lds_fill_rate_probe.jsonl; the matrix units are busy for 7 to 14 %.) Six and eight
// buffers, or requests to registers and stores from there, were 10 to 20 % slower. Two on a CU take
// 0.51 us for a K-tile each, 96 KB through the LDS at 78 bytes per clock of the 263 that the probe's
// mix of requests and reads reaches, the matrix units busy for 18 to 27 %: the same waits.
template <typename E, int TO, bool MUON>
__device__ __forceinline__ void ns_small_body(const NsArgs& args, int step, float ca, float cb,
                                              float cc, const NsMuon& mo) {
  constexpr int T = 64, NI = 2, WT = 32, NB = 4;
  constexpr int OP_BYTES = T * 128, BUF_BYTES = 2 * OP_BYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave8 & 3;
  const bool producer = wave8 >= 4;
  const int wr = wave >> 1, wc = wave & 1;
  NsTile w;
  if (!ns_locate<T, T, TO>(args, step, w)) return;
  f32x4 sum[NI][NI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) sum[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int frow = lane & 15, fq = lane >> 4;
  if (producer) {
    constexpr int R = 2 * NI;                   // requests per wave and K-tile
    unsigned voff_p[NI], voff_q[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = (wave * NI + j) * 8 + (lane >> 3);
      const int kc = (lane & 7) ^ ((row >> 1) & 7);
      const int rp = w.m0 + row < w.M ? row : w.M - 1 - w.m0;
      const int rq = w.n0 + row < w.N ? row : w.N - 1 - w.n0;
      voff_p[j] = 128 * rp + 16 * kc;
      voff_q[j] = 128 * rq + 16 * kc;
    }
    auto request = [&](int kt) {
      char* buf = smem + kt % NB * BUF_BYTES;
      const __amdgpu_buffer_rsrc_t p_rsrc = tile_rsrc(w.P, w.M, w.m0, w.kt0 + kt);
      const __amdgpu_buffer_rsrc_t q_rsrc = tile_rsrc(w.Q, w.N, w.n0, w.kt0 + kt);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int piece = wave * NI + j;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(p_rsrc, (lds_void*)(buf + piece * 1024), 16,
                                                 voff_p[j], 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            q_rsrc, (lds_void*)(buf + OP_BYTES + piece * 1024), 16, voff_q[j], 0, 0, 0);
      }
    };
    for (int kt = 0; kt < NB - 1 && kt < w.nkt; ++kt) request(kt);
    for (int kt = 0; kt < w.nkt; ++kt) {
      // own pieces of K-tile kt have landed; those of up to NB - 2 later ones stay in flight
      if (w.nkt - 1 - kt >= 2)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * R) : "memory");
      else if (w.nkt - 1 - kt == 1)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(R) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_barrier" ::: "memory");
      // behind the barrier the multiplying waves are done with the buffer of K-tile kt - 1
      if (kt + NB - 1 < w.nkt) request(kt + NB - 1);
    }
    asm volatile("s_barrier" ::: "memory");
    if (w.splits == 1) return;
  } else {
    f32x4 acc[NI][NI], cross[NI][NI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) cross[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // fragments of two K-tiles: one is read while the other is multiplied
    f16x8 ph[2][NI], pl[2][NI], qh[2][NI], ql[2][NI];
    auto fetch = [&](int kt, auto odd) {
      constexpr int S = decltype(odd)::value;
      const char* cur = smem + kt % NB * BUF_BYTES;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int rp = wr * WT + i * 16 + frow, rq = wc * WT + i * 16 + frow;
        ql[S][i] = *reinterpret_cast<const f16x8*>(cur + OP_BYTES + piece_off(rq, 4 + fq));
        ph[S][i] = *reinterpret_cast<const f16x8*>(cur + piece_off(rp, fq));
        qh[S][i] = *reinterpret_cast<const f16x8*>(cur + OP_BYTES + piece_off(rq, fq));
        pl[S][i] = *reinterpret_cast<const f16x8*>(cur + piece_off(rp, 4 + fq));
      }
    };
    // one K-tile; FIRST: the accumulators start from zero
    auto multiply = [&](int kt, auto odd, auto first) {
      constexpr int S = decltype(odd)::value;
      constexpr bool FIRST = decltype(first)::value;
      // this K-tile's fragments are here, so its buffer is free behind the barrier; the next
      // K-tile has landed for every wave
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (kt + 1 < w.nkt) {
        asm volatile("s_barrier" ::: "memory");
        if constexpr (S == 0)
          fetch(kt + 1, yes());
        else
          fetch(kt + 1, no());
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          // (operands swapped: a lane's four results lie along N)
          const f32x4 from = FIRST ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[i][j];
          cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[S][j], ph[S][i], cross[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[S][j], ph[S][i], from, 0, 0, 0);
          cross[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[S][j], pl[S][i], cross[i][j], 0, 0, 0);
        }
    };
    asm volatile("s_barrier" ::: "memory");       // K-tile 0 has landed
    fetch(0, no());
    static_assert(NS_CHAIN % 2 == 0, "fragment sets alternate");
    for (int base = 0; base < w.nkt; base += NS_CHAIN) {
      multiply(base, no(), yes());
#pragma unroll
      for (int k = 1; k < NS_CHAIN; k += 2) {
        if (base + k < w.nkt) multiply(base + k, yes(), no());
        if (k + 1 < NS_CHAIN && base + k + 1 < w.nkt) multiply(base + k + 1, no(), no());
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) sum[i][j] += acc[i][j];
    }
    add_cross(sum, cross);
    // the buffers become the epilogue's scratch
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  if (w.splits > 1 && !ns_join<NI, NI, 256>(sum, args, w)) return;
  ns_store<E, NI, NI, TO, MUON>(sum, args, w, step, ca, cb, cc, mo, w.m0 + wr * WT, w.n0 + wc * WT,
                                reinterpret_cast<unsigned*>(smem) + wave * (WT * 36));
}

// 256 x 128 tiles by eight waves of 64 x 64, two per SIMD, one workgroup per CU; three K-tile
// buffers, the requests two K-tiles ahead, one barrier per K-tile.
//
// What bounds it: 8192 x 4096 runs at 1.2 PFLOP/s of matrix work, a library product of 8192^3 in
// fp16 at 1.29. With its matrix instructions alone (registers that do not change) the loop
// reaches 1.54, its LDS-DMA alone would allow 2.0 and its LDS reads alone 4. Three other schedules
// of the same products ended within 3 % of this one: 128 x 128 tiles on two workgroups per CU,
// waves half a K-tile apart (one half reads while the other multiplies), and fragments read ahead
// behind a barrier in the middle of a K-tile. Four waves of 64 x 64 or 128 x 64, one per SIMD, with
// two sets of fragments were 4 to 10 % slower.
template <typename E, int TO, bool MUON>
__device__ __forceinline__ void ns_wide_body(const NsArgs& args, int step, float ca, float cb,
                                             float cc, const NsMuon& mo) {
  constexpr int BM = 256, BN = 128, NI = 4, NB = 3;
  constexpr int P_BYTES = BM * 128, BUF_BYTES = P_BYTES + BN * 128;
  constexpr int RP = 4, RQ = 2, R = RP + RQ;    // requests per wave and K-tile
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 1, wc = wave & 1;
  NsTile w;
  if (!ns_locate<BM, BN, TO>(args, step, w)) return;
  // piece r of an operand: rows 8 (8 r + wave) .. + 7
  unsigned voff_p[RP], voff_q[RQ];
#pragma unroll
  for (int r = 0; r < RP; ++r) {
    const int row = (r * 8 + wave) * 8 + (lane >> 3), kc = (lane & 7) ^ ((row >> 1) & 7);
    voff_p[r] = 128 * (w.m0 + row < w.M ? row : w.M - 1 - w.m0) + 16 * kc;
  }
#pragma unroll
  for (int r = 0; r < RQ; ++r) {
    const int row = (r * 8 + wave) * 8 + (lane >> 3), kc = (lane & 7) ^ ((row >> 1) & 7);
    voff_q[r] = 128 * (w.n0 + row < w.N ? row : w.N - 1 - w.n0) + 16 * kc;
  }
  // (behind the last K-tile the last one again, into a buffer nobody reads: the counts of the
  // waits stay the same)
  auto request = [&](int r, int kt, char* buf) {
    const int at = w.kt0 + (kt < w.nkt ? kt : w.nkt - 1);
    if (r < RP)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(tile_rsrc(w.P, w.M, w.m0, at),
                                               (lds_void*)(buf + (r * 8 + wave) * 1024), 16,
                                               voff_p[r], 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          tile_rsrc(w.Q, w.N, w.n0, at),
          (lds_void*)(buf + P_BYTES + ((r - RP) * 8 + wave) * 1024), 16, voff_q[r - RP], 0, 0, 0);
  };
  const int frow = lane & 15, fq = lane >> 4;
  const int p_hi = piece_off(wr * 64 + frow, fq), p_lo = piece_off(wr * 64 + frow, 4 + fq);
  const int q_hi = P_BYTES + piece_off(wc * 64 + frow, fq);
  const int q_lo = P_BYTES + piece_off(wc * 64 + frow, 4 + fq);
  auto fragment = [&](const char* at, int i) {   // (16 rows further: the same swizzle)
    return *reinterpret_cast<const f16x8*>(at + i * 2048);
  };
  f32x4 sum[NI][NI], acc[NI][NI], cross[NI][NI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) sum[i][j] = cross[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int r = 0; r < R; ++r) request(r, k, smem + k * BUF_BYTES);
  int cur = 0, free = 2 * BUF_BYTES;             // buffers of kt and kt + 2
  // one K-tile; FIRST: the accumulators start from zero
  auto multiply = [&](int kt, auto first) {
    constexpr bool FIRST = decltype(first)::value;
    // every wave's pieces of K-tile kt have landed (those of kt + 1 stay in flight), and every
    // wave is done with the buffer before it
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(R) : "memory");
    const char* buf = smem + cur;
    f16x8 ph[NI], pl[NI], qh[NI], ql[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) ql[j] = fragment(buf + q_lo, j);
    ph[0] = fragment(buf + p_hi, 0);
#pragma unroll
    for (int j = 0; j < NI; ++j) qh[j] = fragment(buf + q_hi, j);
    pl[0] = fragment(buf + p_lo, 0);
    // the order of the instructions is dealt out by hand: behind every four matrix instructions
    // (one of the three products of a row of fragments) the next row's reads or a request
#pragma unroll
    for (int s = 0; s < 3 * NI; ++s) {
      const int i = s / 3, term = s % 3;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        // (operands swapped: a lane's four results lie along N)
        f32x4& to = term == 2 ? acc[i][j] : cross[i][j];
        const f32x4 from = FIRST && term == 2 ? f32x4{0.f, 0.f, 0.f, 0.f} : to;
        to = __builtin_amdgcn_mfma_f32_16x16x32_f16(term == 0 ? ql[j] : qh[j],
                                                    term == 1 ? pl[i] : ph[i], from, 0, 0, 0);
      }
      if (term == 0 && i + 1 < NI) {
        ph[i + 1] = fragment(buf + p_hi, i + 1);
        pl[i + 1] = fragment(buf + p_lo, i + 1);
      }
      if (s % 2 == 1) request(s / 2, kt + 2, smem + free);
      __builtin_amdgcn_sched_barrier(0);
    }
    free = cur;
    cur = cur + BUF_BYTES == NB * BUF_BYTES ? 0 : cur + BUF_BYTES;
  };
  for (int base = 0; base < w.nkt; base += NS_CHAIN) {
    multiply(base, yes());
    const int end = base + NS_CHAIN < w.nkt ? base + NS_CHAIN : w.nkt;
    for (int kt = base + 1; kt < end; ++kt) multiply(kt, no());
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) sum[i][j] += acc[i][j];
  }
  add_cross(sum, cross);
  // the buffers become the epilogue's scratch
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if (w.splits > 1 && !ns_join<NI, NI, 512>(sum, args, w)) return;
  ns_store<E, NI, NI, TO, MUON>(sum, args, w, step, ca, cb, cc, mo, w.m0 + wr * 64, w.n0 + wc * 64,
                                reinterpret_cast<unsigned*>(smem) + wave * (64 * 36));
}

// T = 64: 64 x 64 tiles; 256: 256 x 128
template <typename E, int T, int TO, bool MUON>
__global__ __launch_bounds__(512, T == 64 ? 4 : 2) void ns_product_kernel(
    NsArgs args, int step, float ca, float cb, float cc, NsMuon mo) {
  if constexpr (T == 64)
    ns_small_body<E, TO, MUON>(args, step, ca, cb, cc, mo);
  else
    ns_wide_body<E, TO, MUON>(args, step, ca, cb, cc, mo);
}

#include "newton_schulz_thin.h"
#include "newton_schulz_mid.h"

// ---- host ------------------------------------------------------------------------------------
long up(long v, long to) { return (v + to - 1) / to * to; }

bool is_thin(long rows, long cols) { return (rows < cols ? rows : cols) <= THIN_M; }

// (up to 128 x 2048, as newton_schulz_mid.h says)
bool is_mid(long rows, long cols) {
  const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return !is_thin(rows, cols) && m <= MID_M && n <= MID_N;
}
long mid_slabs(long n) { return (n + MID_SLAB - 1) / MID_SLAB; }

struct NsSizes {
  long m, n, km, kn, parts;
  long slabs, slab_cols;          // thin matrices
  long x, xt, sq;                 // bytes of one image
  long a_parts;                   // of the slabs' parts
  long total;
};
NsSizes sizes_of(long rows, long cols) {
  NsSizes s;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  if (is_thin(rows, cols)) {
    s.slabs = thin_slabs(s.n);
    s.slab_cols = up((s.n + s.slabs - 1) / s.slabs, 16);
    s.total = up(s.slabs * THIN_GRAM * 8, 256);
    return s;
  }
  s.slabs = s.slab_cols = 0;
  s.km = up(s.m, 32);
  s.kn = up(s.n, 32);
  const long want = (rows * cols + 4095) / 4096;
  s.parts = want < NS_MAX_PARTS ? want : NS_MAX_PARTS;
  s.x = up(4 * s.m * s.kn, 256);
  s.xt = up(4 * s.n * s.km, 256);
  s.sq = up(4 * s.m * s.km, 256);
  s.a_parts = is_mid(rows, cols) ? mid_slabs(s.n) * MID_PART : 0;
  s.total = up(8 * s.parts, 256) + s.x + 2 * s.xt + 3 * s.sq + 2 * s.a_parts;
  return s;
}

// (the tile counts of 16 matrices lie within an int)
bool bad_shape(long rows, long cols) {
  return rows < 1 || cols < 1 || rows > 4000000 || cols > 4000000 || rows * cols > (1L << 36);
}

// Sizes of X, A and B over the steps, from the singular values' side: s in [0, r] -> p(s) =
// s q(s^2). The stored fp16 images must hold every entry, and an entry is at most the largest
// singular value. The extremes of p and q lie at the ends and where a quadratic in t = s^2 has
// its roots.
// `factor`: what step k multiplies a singular value by at most.
bool coefficients_fit(int steps, const float* coef, double* factor) {
  double r = 1.0 + 1e-6;
  for (int k = 0; k < steps; ++k) {
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2], end = r * r;
    double p_top = 0.0, q_top = 0.0;
    auto visit = [&](double t) {
      if (!(t >= 0.0 && t <= end)) return;
      const double q = a + b * t + c * t * t;
      p_top = fmax(p_top, fabs(sqrt(t) * q));
      q_top = fmax(q_top, fabs(q));
    };
    if (!(fabs(a) + fabs(b) + fabs(c) < 1e30)) return false;
    visit(0.0);
    visit(end);
    visit(-b / (2.0 * c));                       // q' = 0
    const double root = sqrt(fmax(9.0 * b * b - 20.0 * a * c, 0.0));
    visit((-3.0 * b + root) / (10.0 * c));       // p' = a + 3 b t + 5 c t^2 = 0
    visit((-3.0 * b - root) / (10.0 * c));
    visit(-a / (3.0 * b));                       // ... with c = 0
    if (!(end <= AB_LIMIT) || !(q_top <= AB_LIMIT) || !(p_top <= X_LIMIT)) return false;
    factor[k] = q_top;
    r = p_top * (1.0 + 1e-3);                    // (rounding of what is computed)
  }
  return true;
}

// A tile size: its tiles, the workgroups of a product that run at once, LDS bytes, and by
// measurement what a product takes in us: per launch, for a K-tile in a workgroup that has the chip
// to itself, for a K-tile of the whole chip's work, and for joining split tiles
struct NsShape {
  int bm, bn, slots, lds;
  float launch_us, alone_us, each_us, join_us;
};
NsShape shape_of(int tile) {
  if (tile == 64) return {64, 64, 512, 4 * 2 * 64 * 128, 6.f, 0.23f, 0.0010f, 8.f};
  return {256, 128, 256, 3 * 384 * 128, 14.f, 1.1f, 0.0051f, 24.f};
}
int full_tiles(const NsShape& s, int m, int n) {
  return (m + s.bm - 1) / s.bm * ((n + s.bn - 1) / s.bn);
}
// (row tm of the triangle has bm / bn (tm + 1) tiles; the last row may have fewer columns)
int triangle_tiles(const NsShape& s, int m) {
  const int rows = (m + s.bm - 1) / s.bm, f = s.bm / s.bn;
  return f * rows * (rows + 1) / 2 - (f * rows - (m + s.bn - 1) / s.bn);
}

// Which tiles of a product are split along K: those behind the last full round of the chip, as
// many ways as the round has workgroups for.
void split_rule(const NsShape& shape, int tiles, int kt, int& unsplit, int& splits) {
  unsplit = tiles / shape.slots * shape.slots;
  const int rest = tiles - unsplit, most = rest ? shape.slots / rest : 1;
  splits = split_count(kt, most < 16 ? most : 16);
  if (splits == 1) unsplit = tiles;
}
// us of one product under the split rule: whole rounds of the chip, then what is behind them
float product_us(const NsShape& shape, int tiles, int kt) {
  int unsplit, splits;
  split_rule(shape, tiles, kt, unsplit, splits);
  auto round = [&](int items, int kts) {
    const float one = kts * shape.alone_us, all = (float)items * kts * shape.each_us;
    return items == 0 ? 0.f : one > all ? one : all;
  };
  const int whole = unsplit / shape.slots * shape.slots;
  float us = shape.launch_us + round(whole, kt) + round(unsplit - whole, kt);
  if (splits > 1) us += round((tiles - unsplit) * splits, kt / splits) + shape.join_us;
  return us;
}

// The tile size that takes less time for a product; the wide one where they are close, because it
// takes less power out of what the next product has. Measured (64 x 64 / 256 x 128, us): symmetric
// products of 1024 x 1024 12 / 41, of 2048 x 2048 45 / 54, of 4096 x 4096 312 / 207; full ones of 1024 x
// 1024 by 1024 x 4096 35 / 46, 2048 x 2048 by 2048 x 4096 133 / 98, 4096 x 4096 by 4096 x 8192 1013 / 668.
int faster_tile(const int (&tiles)[2], int kt, float& us) {
  const float small = product_us(shape_of(64), tiles[0], kt);
  const float wide = product_us(shape_of(256), tiles[1], kt);
  us = small <= wide ? small : wide;
  return 1.06f * small <= wide ? 64 : 256;
}

// How a call's tiled matrices are run: in one sequence of launches, or with those of n >= 5/4 m
// in a sequence of their own that takes steps in pairs; and the tile size of each kind of product.
struct NsTiles {
  int gram, square, full;
};
struct NsPlan {
  bool pairs;            // wide matrices apart
  NsTiles tiles[2];      // of the sequence that takes single steps, of the other
};
bool is_wide(long rows, long cols) {
  const long m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return 4 * n >= 5 * m;
}
// us of two steps on the matrices `which` picks (0: all, 1: wide ones, 2: the others)
float steps_us(int count, const int* rows, const int* cols, int which, bool pairs, NsTiles& tiles) {
  int full[2] = {0, 0}, square[2] = {0, 0}, km = 0, kn = 0;
  for (int i = 0; i < count; ++i) {
    if (is_thin(rows[i], cols[i]) || (which && is_wide(rows[i], cols[i]) != (which == 1))) continue;
    const int m = rows[i] < cols[i] ? rows[i] : cols[i], n = rows[i] < cols[i] ? cols[i] : rows[i];
    for (int k = 0; k < 2; ++k) {
      full[k] += full_tiles(shape_of(k ? 256 : 64), m, n);
      square[k] += triangle_tiles(shape_of(k ? 256 : 64), m);
    }
    km = m > km ? m : km;
    kn = n > kn ? n : kn;
  }
  tiles = {64, 64, 64};
  if (!km) return 0.f;
  float g, q, f;
  tiles.gram = faster_tile(square, (kn + 31) / 32, g);
  tiles.square = faster_tile(square, (km + 31) / 32, q);
  tiles.full = faster_tile(full, (km + 31) / 32, f);
  return pairs ? g + 5.f * q + f : 2.f * (g + q + f);
}
NsPlan plan_of(int count, const int* rows, const int* cols) {
  NsPlan one, apart;
  const float whole = steps_us(count, rows, cols, 0, false, one.tiles[0]);
  const float wide = steps_us(count, rows, cols, 1, true, apart.tiles[1]);
  const float rest = steps_us(count, rows, cols, 2, false, apart.tiles[0]);
  one.pairs = false;
  one.tiles[1] = one.tiles[0];
  apart.pairs = true;
  return wide > 0.f && wide + rest < whole ? apart : one;
}

// Steps k and k + 1 taken as one. The second step's A is a polynomial of the first's, so X is
// multiplied twice: A = X X^T, B = q(A), C = B A, A' = C B, B' = q'(A'), P = B' B, X = P X, where
// single steps do it four times. For n = r m that is 3 r + 5 times m^3 instead of 6 r + 2 (2048 x
// 8192 1.71 -> 1.38 ms, 8192 x 4096 6.15 -> 5.33, 1024 x 8192 0.53 -> 0.42). What is lost on A' acts on
// P only through B', beside a I: five steps of 4096 x 8192 are off by 1.7e-6 (single steps 2.1e-6, an
// fp32 computation 5.6e-6), of 1024 x 4096 with a quarter of the rank by 6.5e-6 (5.5e-6, 9.0e-6).
// Three steps as one would lose a^2 as much again. Odd counts have their single step before the
// last pair, where the singular values are least apart. P has to fit the images of B.
bool step_pairs(int k, int steps, const double* factor) {
  if (k + 1 >= steps || ((steps - k) % 2 && k + 3 >= steps)) return false;
  return factor[k] * factor[k + 1] <= AB_LIMIT;
}

// matrices that go through the same launches
struct NsSet {
  NsArgs args;
  NsTiles tiles;
  bool pairs;
};

// One kind of product of a set: its tiles, and the launch of them
struct NsLaunch {
  NsArgs args;
  NsShape shape;
  template <typename Tiles>                      // tiles(shape, matrix)
  NsLaunch(const NsSet& set, int tile, int kt_max, Tiles tiles)
      : args(set.args), shape(shape_of(tile)) {
    for (int i = 0; i < args.count; ++i) args.first[i + 1] = args.first[i] + tiles(shape, args.t[i]);
    split_rule(shape, args.first[args.count], kt_max, args.unsplit, args.splits);
  }
  template <typename E, int TO, bool MUON>
  void run(int p, int q, int to, int turn, const float* c, const NsMuon& mo, hipStream_t stream) {
    args.p = p;
    args.q = q;
    args.to = to;
    const unsigned grid =
        args.unsplit + (args.first[args.count] - args.unsplit) * (unsigned)args.splits;
    if (shape.bm == 64)
      hipLaunchKernelGGL((ns_product_kernel<E, 64, TO, MUON>), dim3(grid), dim3(512), shape.lds,
                         stream, args, turn, c[0], c[1], c[2], mo);
    else
      hipLaunchKernelGGL((ns_product_kernel<E, 256, TO, MUON>), dim3(grid), dim3(512), shape.lds,
                         stream, args, turn, c[0], c[1], c[2], mo);
  }
};

template <typename E, int T, bool MUON>
void allow_product_lds() {
  const int lds = shape_of(T).lds;
  allow_lds(ns_product_kernel<float, T, TO_A, false>, lds);
  allow_lds(ns_product_kernel<float, T, TO_B, false>, lds);
  allow_lds(ns_product_kernel<float, T, TO_S, false>, lds);
  allow_lds(ns_product_kernel<float, T, TO_X, false>, lds);
  allow_lds(ns_product_kernel<E, T, TO_OUT, MUON>, lds);
}

template <typename E, bool MUON>
int launch_steps(const NsSet& set, int steps, const float* coef, const double* factor,
                 const NsMuon& mo, hipStream_t stream) {
  static DtfPerDeviceOnce once;
  dtf_once_per_device(once, [] {
    allow_product_lds<E, 64, MUON>();
    allow_product_lds<E, 256, MUON>();
  });
  int km = 0, kn = 0;
  for (int i = 0; i < set.args.count; ++i) {
    const NsMat& t = set.args.t[i];
    km = t.km > km ? t.km : km;
    kn = t.kn > kn ? t.kn : kn;
  }
  const auto triangle = [](const NsShape& s, const NsMat& t) { return triangle_tiles(s, t.m); };
  NsLaunch gram(set, set.tiles.gram, kn / 32, triangle);
  NsLaunch square(set, set.tiles.square, km / 32, triangle);
  NsLaunch full(set, set.tiles.full, km / 32,
                [](const NsShape& s, const NsMat& t) { return full_tiles(s, t.m, t.n); });
  // (the last product's tiles lie along the caller's rows)
  NsLaunch last(set, set.tiles.full, km / 32,
                [](const NsShape& s, const NsMat& t) { return full_tiles(s, t.rows, t.cols); });
  for (int k = 0, turn = 0; k < steps; ++turn) {
    const float* c = coef + 3 * k;
    int at = 1;                                                                // factor of X
    gram.run<float, TO_A, false>(0, 0, 0, turn, c, mo, stream);                // A
    square.run<float, TO_B, false>(0, 0, 1, turn, c, mo, stream);              // B
    if (set.pairs && step_pairs(k, steps, factor)) {
      square.run<float, TO_S, false>(1, 0, 2, turn, c, mo, stream);            // C = B A
      square.run<float, TO_S, false>(2, 1, 0, turn, c, mo, stream);            // A' = C B
      square.run<float, TO_B, false>(0, 0, 2, turn, c + 3, mo, stream);        // B'
      square.run<float, TO_S, false>(2, 1, 0, turn, c, mo, stream);            // P = B' B
      at = 0;
      ++k;
    }
    if (++k < steps)
      full.run<float, TO_X, false>(at, 0, 0, turn, c, mo, stream);
    else
      last.run<E, TO_OUT, MUON>(at, 0, 0, turn, c, mo, stream);
  }
  DTF_LAUNCH_CHECK();
  return DTF_OK;
}

// The whole call in launches of one or two steps (newton_schulz_mid.h)
template <int KT, typename E, bool MUON>
int launch_mid(const NsArgs& args, int steps, const float* coef, const double* factor, float eps,
               const NsMuon& mo, hipStream_t stream) {
  constexpr int LDS = 2 * MID_MAT;
  static DtfPerDeviceOnce once;
  dtf_once_per_device(once, [&] {
    allow_lds(ns_mid_kernel<KT, E, MID_FIRST, MUON>, LDS);
    allow_lds(ns_mid_kernel<KT, float, MID_STEP, false>, LDS);
    allow_lds(ns_mid_kernel<KT, E, MID_LAST, MUON>, LDS);
  });
  MidArgs now = {};
  now.count = args.count;
  for (int i = 0; i < args.count; ++i) {
    now.t[i] = args.t[i];
    now.first[i + 1] = now.first[i] + (int)mid_slabs(args.t[i].n);
  }
  const dim3 grid(now.first[now.count]), block(MID_THREADS);
  hipLaunchKernelGGL((ns_mid_kernel<KT, E, MID_FIRST, MUON>), grid, block, LDS, stream, now, eps, mo);
  for (int k = 0; k < steps;) {
    now.pair = step_pairs(k, steps, factor);
    ++now.turn;
    for (int i = 0; i < 3 + 3 * now.pair; ++i) now.c[i] = coef[3 * k + i];
    k += 1 + now.pair;
    if (k < steps)
      hipLaunchKernelGGL((ns_mid_kernel<KT, float, MID_STEP, false>), grid, block, LDS, stream, now,
                         eps, mo);
    else
      hipLaunchKernelGGL((ns_mid_kernel<KT, E, MID_LAST, MUON>), grid, block, LDS, stream, now, eps,
                         mo);
  }
  DTF_LAUNCH_CHECK();
  return DTF_OK;
}

// head of the workspace: arrival counts, then the partial tiles of one split product
constexpr long NS_HEAD = 4L * NS_SLOTS;
long shared_bytes(const NsPlan& plan) {
  bool wide = false;
  for (const NsTiles& t : plan.tiles)
    wide = wide || t.gram != 64 || t.square != 64 || t.full != 64;
  const NsShape s = shape_of(wide ? 256 : 64);
  return NS_HEAD + 4L * s.slots * s.bm * s.bn;
}

template <typename E, bool MUON>
int launch(const NsSet (&sets)[2], const NsArgs& parts, const NsArgs& split, const NsArgs& thin,
           int steps, const float* coef, const double* factor, float eps, const NsMuon& mo,
           hipStream_t stream) {
  if (thin.count) {
    const int rc = launch_thin<E, MUON>(thin, steps, coef, eps, mo, stream);
    if (rc != DTF_OK) return rc;
  }
  const int n = parts.count;
  if (n == 0) return DTF_OK;
  hipLaunchKernelGGL((ns_norm_kernel<E, MUON>), dim3(parts.first[n]), dim3(256), 0, stream, parts,
                     mo);
  DTF_LAUNCH_CHECK();
  bool mid = true;
  int m = 0;
  for (int i = 0; i < n; ++i) {
    mid = mid && is_mid(parts.t[i].rows, parts.t[i].cols);
    m = parts.t[i].m > m ? parts.t[i].m : m;
  }
  if (mid && m <= 96) return launch_mid<3, E, MUON>(parts, steps, coef, factor, eps, mo, stream);
  if (mid) return launch_mid<4, E, MUON>(parts, steps, coef, factor, eps, mo, stream);
  hipLaunchKernelGGL((ns_split_kernel<E, MUON>), dim3(split.first[n]), dim3(256), 0, stream, split,
                     eps, mo);
  DTF_LAUNCH_CHECK();
  for (const NsSet& set : sets) {
    if (set.args.count == 0) continue;
    const int rc = launch_steps<E, MUON>(set, steps, coef, factor, mo, stream);
    if (rc != DTF_OK) return rc;
  }
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
  double factor[NS_MAX_STEPS];
  if (!coefficients_fit(steps, coef, factor)) return DTF_ERR_UNSUPPORTED;
  // thin matrices have kernels of their own; the others share the tiled sequence
  NsArgs args = {}, thin = {};
  char* at = (char*)workspace;
  if ((uintptr_t)at & 255) return DTF_ERR_BAD_ARG;
  long used = 0;
  bool tiled = false;
  for (int i = 0; i < count; ++i) {
    if (bad_shape(rows[i], cols[i])) return DTF_ERR_BAD_ARG;
    tiled = tiled || !is_thin(rows[i], cols[i]);
  }
  const NsPlan plan = plan_of(count, rows, cols);
  if (tiled) {
    args.arrived = (int*)at;
    args.partial = (float*)(at + NS_HEAD);
    used = shared_bytes(plan);
    at += used;
  }
  for (int i = 0; i < count; ++i) {
    if (!g[i] || !out[i] || (MUON && (!v[i]))) return DTF_ERR_BAD_ARG;
    const NsSizes s = sizes_of(rows[i], cols[i]);
    NsArgs& to = s.slabs ? thin : args;
    NsMat& t = to.t[to.count++];
    t.g = g[i];
    t.out = out[i];
    t.v = MUON ? v[i] : nullptr;
    t.scale = MUON ? scale[i] : 1.f;
    t.rows = rows[i];
    t.cols = cols[i];
    t.m = (int)s.m;
    t.n = (int)s.n;
    used += s.total;
    if (used > workspace_bytes) return DTF_ERR_BAD_ARG;
    if (s.slabs) {
      t.gram = (double*)at;
      t.slabs = (int)s.slabs;
      t.slab_cols = (int)s.slab_cols;
      at += s.total;
      continue;
    }
    t.km = (int)s.km;
    t.kn = (int)s.kn;
    t.nparts = (int)s.parts;
    t.parts = (double*)at;
    at += up(8 * s.parts, 256);
    t.x = at;
    at += s.x;
    t.xt0 = at;
    at += s.xt;
    t.xt1 = at;
    at += s.xt;
    for (char*& sq : t.sq) {
      sq = at;
      at += s.sq;
    }
    for (char*& a : t.a_parts) {
      a = at;
      at += s.a_parts;
    }
  }
  NsArgs parts = args, split = args;
  for (int i = 0; i < args.count; ++i) {
    const NsMat& t = args.t[i];
    const long tiles = ((t.rows + 63L) / 64) * ((t.cols + 63L) / 64);
    if (split.first[i] + tiles > (1L << 30)) return DTF_ERR_UNSUPPORTED;
    parts.first[i + 1] = parts.first[i] + t.nparts;
    split.first[i + 1] = split.first[i] + (int)tiles;
  }
  NsSet sets[2] = {{args, plan.tiles[0], false}, {args, plan.tiles[1], true}};
  sets[0].args.count = sets[1].args.count = 0;
  for (int i = 0; i < args.count; ++i) {
    NsArgs& to = sets[plan.pairs && is_wide(args.t[i].rows, args.t[i].cols)].args;
    to.t[to.count++] = args.t[i];
  }
  switch (type) {
    case NS_F32:
      return launch<float, MUON>(sets, parts, split, thin, steps, coef, factor, eps, mo, stream);
    case NS_BF16:
      if constexpr (!MUON)
        return launch<dtf_bf16, false>(sets, parts, split, thin, steps, coef, factor, eps, mo, stream);
      break;
    default:
      if constexpr (!MUON)
        return launch<_Float16, false>(sets, parts, split, thin, steps, coef, factor, eps, mo, stream);
      break;
  }
  return DTF_ERR_BAD_ARG;
}

}  // namespace

// bytes of workspace (256-byte aligned) for `count` matrices; 0 for shapes that are not taken
DTF_API long dtf_newton_schulz_workspace(int count, const int* rows, const int* cols) {
  if (count < 0 || count > NS_MAX_MATS || (count > 0 && (!rows || !cols))) return 0;
  long total = 256;
  bool tiled = false;
  for (int i = 0; i < count; ++i) {
    if (bad_shape(rows[i], cols[i])) return 0;
    tiled = tiled || !is_thin(rows[i], cols[i]);
    total += sizes_of(rows[i], cols[i]).total;
  }
  return total + (tiled ? shared_bytes(plan_of(count, rows, cols)) : 0);
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
