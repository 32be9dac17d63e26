// Muon's update of weight matrices: the momentum, its orthogonalisation by Newton-Schulz products, the weights.
//
//   m <- m + (1 - mu)(g - m),  u = g + mu (m - g) (Nesterov) or m             (g clipped by its group's norm)
//   X = u / max(|u|_F, eps)                                                     on the side with fewer rows: r <= c
//   X <- a X + (b A + c A A) X,  A = X X^T                                      `steps` times
//   p <- decay p - lr scale X
//
// Three products a step: A = X X^T from the rows of X; A A from the rows of A, which is symmetric; B X, B = b A + c A A,
// from the rows of B and, by transposing LDS loads, the rows of X.  So X is kept in one order only.  A and B are
// symmetric: only tiles on or below the diagonal are computed, the others are written as mirrors -- 3 r^2 c + r^3
// floating-point operations a step in place of 4 r^2 c + 2 r^3.
//
// What bounds it.  Large matrices: the products, at the rate the card's power allows (4096 x 4096: prec 0, three products
// for one, 3.27 .. 3.45 ms, 1190 .. 1260 TFLOP/s of its fp16 products; prec 1 1.34 .. 1.46 ms, 940 .. 1025; a library
// product reaches 1040 .. 1110 at that size, 1308 at 8192; a 2048-wide block of six matrices, prec 0: 4.34 .. 4.56 ms,
// 975 .. 1025).
// Stacks of 1024 x 4096: the iterates' way through memory beside them (prec 1: 8 bytes an element and step, with the
// operand 10).  Small ones: 2 + 3 steps launches of 4 to 8 us, each one block's loads, products and stores in a row (the
// renderer's 19 matrices: 131 us).
//
// Precision.  Operands are fp16, X, A and B each times the largest power of two that its entries allow: they are bounded
// by singular values, those by the coefficients (2^15 X, 2^15 A, 2^14 B for a, b, c = 3.4445, -4.7750, 2.0315); fp32
// accumulators.
//   prec 0  x = hi + 2^-6 lo, both fp16; a product is hi hi + 2^-6 (hi lo + lo hi): as near the definition as fp32
//           products, at a third of the fp16 matrix rate (fp32 MFMA: a sixteenth).  Entries of X from 2^-23 on -- a
//           gradient's from 2^-23 of its norm -- keep 22 bits, smaller ones are within 2^-46.  So the small part of an
//           uneven gradient keeps its accuracy too: noise beside an entry of 10^6 is 1.2e-7 off (with lo itself in fp16
//           and a unit of 2^10 for all: 1.8e-5; float32 products 0.8e-7).  bf16 pairs hold 16 bits only, which the
//           map's slope (up to a^5 = 485 for small singular values) takes to 3e-5 .. 2e-4.
//   prec 1  one fp16 product.  X itself keeps hi + lo and a X is added from those in fp32: rounding only enters
//           through (b A + c A A) X, so the result is 0.6e-3 .. 1.6e-3 off, under bf16's own 1.7e-3 (3e-3 where one
//           entry stands for nearly all of the norm; X rounded to fp16 between steps: up to 1.2e-2 where a few
//           directions are far stronger than the rest).  Matrices of up to 128
//           rows or columns run prec 0 all the same: they wait for launches and loads, not for products, and with few
//           entries to average over, single products are up to 3.8e-3 off.
//
// Every matrix of a call takes part in the same 2 + 3 steps launches; a block finds its matrix and tile by blockIdx.
// Operands are padded to 64 rows and columns, with zeros, and what a wider tile has past them is never stored, so the
// product loop has no bounds checks.
#include "common.h"
#include "chain_common.h"

#include <algorithm>
#include <new>
#include <type_traits>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
// pointers read from a table are generic to the compiler (flat loads and stores): these are to device memory
#define MMS_GLOBAL __attribute__((address_space(1)))
typedef MMS_GLOBAL char gchar;
typedef MMS_GLOBAL _Float16 ghalf;
typedef MMS_GLOBAL half4 ghalf4;
typedef MMS_GLOBAL half8 ghalf8;
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

constexpr int kMaxMatrices = 4096;       // (or stacks) per call
constexpr int kNsItems = 48;             // matrices (or stacks of them) per launch: the argument struct stays < 4 KB
constexpr float kLow = 64.f;             // what hi leaves of a value is held 2^6 times
constexpr float kUnlow = 1.f / 64.f;
constexpr float kHalfMax = 60000.f;      // fp16's largest value, less a margin for roundings
constexpr int kNormBlocks = 1024;        // blocks per matrix that sum squares, at most
constexpr int kNormElems = 8192;         // elements per such block, at least
constexpr int64_t kMaxBlocks = 1 << 23;  // of a launch (times its threads: below 2^32)

struct NsItem {
  const void* g;       // gradient (or the matrix to orthogonalise)
  float* m;            // momentum [batch, rows, cols], or null
  void* p;             // weights (or the result)
  char* ws;            // this item's part of the workspace
  int64_t bsg, bsp;    // elements between the matrices of a stack
  int ldg, ldp;
  int rows, cols, batch;
  float scale;         // of the learning rate
};

struct NsArgs {
  int n;
  int blk0[kNsItems + 1];   // first block of each item
  NsItem it[kNsItems];
};

// The items again, in the workspace: written by the first launch, read by the others.  (Kernel arguments lie in host
// memory: 3.6 KB of them cost each launch several us on the host, and each block a slow read.)
constexpr int kMaxParts = 1024;   // blocks of a launch of A whose tiles are summed in parts
struct NsTable {
  int blk0[4][64];          // first block of each item: packing, A, B, X; INT_MAX past the last
  NsItem it[kNsItems];
  int arrived[kMaxParts];   // parts of a tile of A that are through; zero between launches
};
constexpr int64_t kTableBytes = 8704;
static_assert(sizeof(NsTable) <= kTableBytes, "the table's part of the workspace");
enum { MAP_PACK = 0, MAP_A = 1, MAP_B = 2, MAP_X = 3 };
struct NsTiles {
  int a, b, x;
  int chunk;   // stages of A that a block sums, at most
};

struct NsStep {
  float momentum, rest;     // mu and 1 - mu, each rounded once (1 - 0.95f is 2e-7 off)
  int nesterov;
  const float* sumsq;       // of the whole gradient, or null: no clipping
  float max_norm;
  const float* hyper;       // device [decay, -lr], or null: the two values
  float decay, neg_lr;
  double eps;
  float unit[3];            // fp16 operands hold X, A and B = b A + c A A times these powers of two
};

// The workspace of one matrix: norm partials, then the fp16 operands.  W: 2 with hi and lo (32 of each in turn along
// k, so that a 128-byte line holds both), 1 with hi only.
struct NsLayout {
  int rp, cp, w;
  __host__ __device__ NsLayout(int rows, int cols, int w_) : w(w_) {
    const int r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
    rp = (r + 63) / 64 * 64;
    cp = (c + 63) / 64 * 64;
  }
  __host__ __device__ int64_t x(int i) const { return kNormBlocks * (int64_t)sizeof(double) + (int64_t)rp * cp * w * 2 * i; }
  __host__ __device__ int64_t a() const { return x(2); }
  __host__ __device__ int64_t b() const { return a() + (int64_t)rp * rp * w * 2; }
  __host__ __device__ int64_t xlo() const { return b() + (int64_t)rp * rp * w * 2; }
  __host__ __device__ int64_t bytes() const { return xlo() + (w == 1 ? (int64_t)rp * cp * 2 : 0); }
};

// the item of a block: every lane compares one item's first block (one load; a search through the arguments, which lie
// in host memory, waits for each of its steps)
__device__ __forceinline__ int find_item(const NsArgs& A, int blk) {
  const int lane = threadIdx.x & 63;
  const bool before = lane < A.n && A.blk0[lane < kNsItems ? lane : 0] <= blk;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
}
__device__ __forceinline__ int find_item(const NsTable* T, int map, int& first) {
  const int blk = blockIdx.x, b0 = T->blk0[map][threadIdx.x & 63];
  const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(b0 <= blk)) - 1);
  first = __builtin_amdgcn_readlane(b0, i);
  return i;
}
// the item by scalar loads (nothing writes the table while this launch runs)
__device__ __forceinline__ NsItem load_item(const NsTable* T, int i) {
  typedef const __attribute__((address_space(4))) uint64_t* words;
  const words src = (words)(uintptr_t)(T->it + i);
  static_assert(sizeof(NsItem) % 8 == 0, "whole words");
  uint64_t w[sizeof(NsItem) / 8];
#pragma unroll
  for (size_t q = 0; q < sizeof(NsItem) / 8; ++q) w[q] = src[q];
  return __builtin_bit_cast(NsItem, w);
}

// blocks of a matrix in each launch
__host__ __device__ inline int norm_blocks(int64_t rows, int64_t cols) {
  const int64_t nb = (rows * cols + kNormElems - 1) / kNormElems;
  return nb < 1 ? 1 : nb > kNormBlocks ? kNormBlocks : (int)nb;
}
__host__ __device__ inline int pack_blocks(const NsLayout& L) { return (L.rp / 64) * (L.cp / 64); }
__host__ __device__ inline int gram_blocks(const NsLayout& L, int tile) {
  const int n = (L.rp + tile - 1) / tile;
  return n * (n + 1) / 2;
}
__host__ __device__ inline int full_blocks(const NsLayout& L, int tile) {
  return ((L.rp + tile - 1) / tile) * ((L.cp + tile - 1) / tile);
}

// blocks that share the sum of a tile of A, each over `chunk` stages of 128 bytes along k
__host__ __device__ inline int gram_parts(const NsLayout& L, int chunk) { return (L.cp * L.w / 64 + chunk - 1) / chunk; }

__device__ __forceinline__ float load1(const MMS_GLOBAL void* p, int64_t i, bool bf16) {
  if (bf16) return __uint_as_float((uint32_t)((const MMS_GLOBAL uint16_t*)p)[i] << 16);
  return ((const MMS_GLOBAL float*)p)[i];
}
__device__ __forceinline__ uint16_t to_bf16(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ void store1(MMS_GLOBAL void* p, int64_t i, bool bf16, float v) {
  if (bf16) ((MMS_GLOBAL uint16_t*)p)[i] = to_bf16(v);
  else ((MMS_GLOBAL float*)p)[i] = v;
}

__device__ __forceinline__ float clip_of(const NsStep& s) {
  if (!s.sumsq) return 1.f;
  const float c = s.max_norm / (sqrtf(s.sumsq[0]) + 1e-6f);
  return c < 1.f ? c : 1.f;
}

// ---- momentum and the sum of squares ----------------------------------------------------------------------------
// Reads g and m, writes m (12 bytes an element in fp32), and leaves each block's sum of u^2, in double: gradients of
// 1e-25 or 1e25 keep their norm.  u is not stored: the next launch forms it again from the g and m it has to read.
__global__ __launch_bounds__(256) void muon_momentum_kernel(NsArgs A, NsStep S, int bf16, int w, NsTiles tiles,
                                                            NsTable* __restrict__ table) {
  __shared__ double red[4];
  if (blockIdx.x == 0 && threadIdx.x < 64) {
    const int i = threadIdx.x, k = i < A.n ? i : 0;
    const NsItem it = A.it[k];
    const NsLayout L(it.rows, it.cols, w);
    const int count[4] = {pack_blocks(L) * it.batch, gram_blocks(L, tiles.a) * gram_parts(L, tiles.chunk) * it.batch,
                          gram_blocks(L, tiles.b) * it.batch, full_blocks(L, tiles.x) * it.batch};
    for (int q = 0; q < 4; ++q) {
      int x = i < A.n ? count[q] : 0;
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (i >= o) x += y;
      }
      table->blk0[q][i] = i < A.n ? x - count[q] : 0x7fffffff;
    }
    if (i < A.n) table->it[i] = it;
  }
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < kMaxParts; i += 256) table->arrived[i] = 0;
  const int ii = find_item(A, blockIdx.x);
  const NsItem it = A.it[ii];
  const NsLayout L(it.rows, it.cols, w);
  const int per = (A.blk0[ii + 1] - A.blk0[ii]) / it.batch;
  const int k = (blockIdx.x - A.blk0[ii]) / per, b = (blockIdx.x - A.blk0[ii]) % per;
  const int64_t n = (int64_t)it.rows * it.cols;
  const gchar* g = (const gchar*)it.g + k * it.bsg * (bf16 ? 2 : 4);
  MMS_GLOBAL float* m = it.m ? (MMS_GLOBAL float*)it.m + k * n : nullptr;
  const float clip = clip_of(S), w1 = S.rest, mu = S.momentum;
  double sum = 0.0;
  const auto one = [&](int64_t i, float gi, float& mi) {
    gi *= clip;
    float u = gi;
    if (m) {
      mi = __builtin_fmaf(w1, gi - mi, mi);
      u = S.nesterov ? __builtin_fmaf(mu, mi - gi, gi) : mi;
    }
    sum += (double)u * u;
  };
  const bool dense = it.ldg == it.cols;
  const int64_t step = (int64_t)per * 256;
  if (dense && n % 4 == 0 && ((uint64_t)g & (bf16 ? 7 : 15)) == 0 && ((uint64_t)m & 15) == 0) {
    for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n / 4; i += step) {
      float gi[4];
      if (bf16) {
        const uint2 q = *(const uint2*)((const char*)g + 8 * i);
        gi[0] = __uint_as_float(q.x << 16); gi[1] = __uint_as_float(q.x & 0xffff0000u);
        gi[2] = __uint_as_float(q.y << 16); gi[3] = __uint_as_float(q.y & 0xffff0000u);
      } else {
        const float4 q = *(const float4*)((const char*)g + 16 * i);
        gi[0] = q.x; gi[1] = q.y; gi[2] = q.z; gi[3] = q.w;
      }
      float4 mi = m ? *(const float4*)((const float*)m + 4 * i) : float4{0.f, 0.f, 0.f, 0.f};
      one(4 * i, gi[0], mi.x); one(4 * i + 1, gi[1], mi.y); one(4 * i + 2, gi[2], mi.z); one(4 * i + 3, gi[3], mi.w);
      if (m) *(float4*)((float*)m + 4 * i) = mi;
    }
  } else {
    for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n; i += step) {
      float mi = m ? m[i] : 0.f;
      one(i, load1(g, dense ? i : (i / it.cols) * it.ldg + i % it.cols, bf16), mi);
      if (m) m[i] = mi;
    }
  }
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) ((double*)(it.ws + k * L.bytes()))[b] = red[0] + red[1] + red[2] + red[3];
}

// Position of (row, k) in an operand of R rows: 32 columns at a time, all rows of them one after another, so that a
// stage of a tile is one contiguous piece (rows of a power of two of bytes apart would meet in few of the L2's
// channels).  With hi and lo, a row holds 32 of each.
template <int W>
__device__ __forceinline__ int64_t at(int row, int R, int k) {
  return ((int64_t)(k >> 5) * R + row) * (32 * W) + (k & 31);
}

template <int N>
__device__ __forceinline__ void split_n(const float* v, _Float16* hi, _Float16* lo) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    hi[q] = (_Float16)v[q];
    lo[q] = (_Float16)((v[q] - (float)hi[q]) * kLow);
  }
}

// ---- X of u / |u| -------------------------------------------------------------------------------------------------
// One 64 x 64 tile of u per block through LDS, written on the side with fewer rows; the padding as zeros.
template <int W>
__global__ __launch_bounds__(256) void ns_pack_kernel(const NsTable* __restrict__ T, NsStep S, int bf16) {
  __shared__ float t[64][65];
  __shared__ double red[4];
  int first;
  const NsItem it = load_item(T, find_item(T, MAP_PACK, first));
  const NsLayout L(it.rows, it.cols, W);
  const bool tall = it.rows > it.cols;
  const int tr = (tall ? L.cp : L.rp) / 64, tc = (tall ? L.rp : L.cp) / 64;
  const int q = blockIdx.x - first;
  const int k = q / (tr * tc), i0 = (q / tc) % tr * 64, j0 = q % tc * 64;
  gchar* ws = (gchar*)it.ws + k * L.bytes();
  const int64_t n = (int64_t)it.rows * it.cols;
  const gchar* g = (const gchar*)it.g + k * it.bsg * (bf16 ? 2 : 4);
  const MMS_GLOBAL float* m = it.m ? (const MMS_GLOBAL float*)it.m + k * n : nullptr;
  const float clip = clip_of(S), mu = S.momentum;
  // u, 16 values a thread: 4 columns of 4 rows, or 1 of 16 where rows are not whole 16 bytes (8 of bf16)
  float gv[16], mv[16];
  const bool quads = it.cols % 4 == 0 && it.ldg % 4 == 0 && ((uint64_t)g & (bf16 ? 7 : 15)) == 0 && ((uint64_t)m & 15) == 0;
  const int lane16 = threadIdx.x & 15, lane64 = threadIdx.x & 63;
#pragma unroll
  for (int e = 0; e < 16; ++e) gv[e] = mv[e] = 0.f;
  if (quads) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * 16 + (threadIdx.x >> 4), j = j0 + lane16 * 4;
      if (i < it.rows && j < it.cols) {
        const int64_t at = (int64_t)i * it.ldg + j;
        if (bf16) {
          const uint64_t v = *(const MMS_GLOBAL uint64_t*)(g + at * 2);
#pragma unroll
          for (int z = 0; z < 4; ++z) gv[e * 4 + z] = __uint_as_float((uint32_t)(v >> (16 * z)) << 16);
        } else {
          const floatx4 v = *(const MMS_GLOBAL floatx4*)(g + at * 4);
#pragma unroll
          for (int z = 0; z < 4; ++z) gv[e * 4 + z] = v[z];
        }
        if (m) {
          const floatx4 v = *(const MMS_GLOBAL floatx4*)(m + (int64_t)i * it.cols + j);
#pragma unroll
          for (int z = 0; z < 4; ++z) mv[e * 4 + z] = v[z];
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int i = i0 + e * 4 + (threadIdx.x >> 6), j = j0 + lane64;
      if (i < it.rows && j < it.cols) {
        gv[e] = load1(g, (int64_t)i * it.ldg + j, bf16);
        if (m) mv[e] = m[(int64_t)i * it.cols + j];
      }
    }
  }
  // |u|: the partial sums in a fixed order
  const int nb = norm_blocks(it.rows, it.cols);
  double sum = 0.0;
  for (int i = threadIdx.x; i < nb; i += 256) sum += ((const MMS_GLOBAL double*)ws)[i];
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  norm = norm < S.eps ? S.eps : norm;
  const double inv = (double)S.unit[0] / norm;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float gi = gv[e] * clip;
    const float u = !m ? gi : S.nesterov ? __builtin_fmaf(mu, mv[e] - gi, gi) : mv[e];
    const int i = quads ? (e >> 2) * 16 + (threadIdx.x >> 4) : e * 4 + (threadIdx.x >> 6);
    t[i][quads ? lane16 * 4 + (e & 3) : lane64] = (float)(u * inv);
  }
  __syncthreads();
  ghalf* X = (ghalf*)(ws + L.x(0));
  ghalf* Xlo = (ghalf*)(ws + L.xlo());
  const int x0 = tall ? j0 : i0, y0 = tall ? i0 : j0;
  for (int e = threadIdx.x; e < 64 * 16; e += 256) {
    const int a = (e >> 3) & 63, b = (e >> 9) * 32 + (e & 7) * 4;   // 8 threads: the 32 columns of a row; then rows
    half4 hi, lo;
    float v[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) v[z] = tall ? t[b + z][a] : t[a][b + z];
    split_n<4>(v, (_Float16*)&hi, (_Float16*)&lo);
    const int64_t d = at<W>(x0 + a, L.rp, y0 + b);
    *(ghalf4*)(X + d) = hi;
    *(ghalf4*)(W == 2 ? X + d + 32 : Xlo + d) = lo;
  }
}

// ---- the products -------------------------------------------------------------------------------------------------
enum { PHASE_A = 0, PHASE_B = 1, PHASE_X = 2, PHASE_LAST = 3 };

// 16 bytes per lane, global -> LDS: scalar base and 32-bit offset per lane
__device__ __forceinline__ void lds_dma16_s(const char* base, uint32_t off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_addr)
               : "memory", "m0");
}

// a pointer that every lane holds alike, in scalar registers
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// One TILE x TILE tile of P Q^T per block.  WM x WN: a wave's part.  A stage is 128 bytes of every row (64 values, or 32
// hi and 32 lo), brought to LDS by DMA; the 16-byte chunk c of row i lies at c ^ (i & 7), which makes the fragment reads
// (8 lanes = 8 rows, one chunk) free of bank conflicts.  NBUF stages form a ring, NBUF - 1 of them in flight.
//
// The product with X has X's rows along k: a stage of it is 64 (32) rows of the tile's columns, 4 KB for each 32 columns,
// and its fragments are read by the transposing LDS loads: 16 lanes read 4 rows of 16 columns, and each gets one column
// of them.  There a row's 32-byte piece lies at piece ^ f(row), f by bit 3 of the row (and bit 1 where rows are 128
// bytes): the 8 rows that 32 lanes read are in different banks.  So X^T is kept nowhere.
template <int TILE, int WM, int WN, int NBUF, int W, int PHASE>
__global__ __launch_bounds__((TILE / WM) * (TILE / WN) * 64) void ns_product_kernel(
    NsTable* __restrict__ T, NsStep S, float mul, float ca, float cb, float cc, int parity, int bf16, int chunk,
    uint64_t* __restrict__ partial) {
  constexpr int NWM = TILE / WM, NWN = TILE / WN, NW = NWM * NWN, NT = NW * 64;
  constexpr int STAGE = 2 * TILE * 128;          // bytes
  constexpr int LOADS = STAGE / (NW * 1024);     // DMA instructions per wave and stage, 8 rows each
  constexpr int FM = WM / 16, FN = WN / 16;
  constexpr int SLAB = 64 * (TILE + 1) * 4;
  __shared__ __attribute__((aligned(1024))) char lds[NBUF * STAGE > SLAB ? NBUF * STAGE : SLAB];

  int first;
  const NsItem it = load_item(T, find_item(T, PHASE == PHASE_A ? MAP_A : PHASE == PHASE_B ? MAP_B : MAP_X, first));
  const NsLayout L(it.rows, it.cols, W);
  const int nr = (L.rp + TILE - 1) / TILE, nc = (L.cp + TILE - 1) / TILE;
  const int tiles = PHASE <= PHASE_B ? nr * (nr + 1) / 2 : nr * nc;
  const int parts = PHASE == PHASE_A ? __builtin_amdgcn_readfirstlane(gram_parts(L, chunk)) : 1, per = tiles * parts;
  int q = blockIdx.x - first, ti, tj;
  {
    // blocks b, b + 8, ... share an XCD: give each XCD a run of neighbouring tiles of the item
    const int o = first & 7, x = (q + o) & 7, last = per * it.batch + o - 1;
    int start = 0;
    for (int y = 0; y < x; ++y) start += (last - y >= 0 ? ((last - y) >> 3) + 1 : 0) - (y < o ? 1 : 0);
    q = start + ((q + o) >> 3) - (x < o ? 1 : 0);
  }
  const int k = q / per, slot = first + q;
  q -= k * per;
  const int part = PHASE == PHASE_A ? __builtin_amdgcn_readfirstlane(q / tiles) : 0;
  q -= part * tiles;
  if (PHASE <= PHASE_B) {
    ti = (int)((sqrtf(8.f * q + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= q) ++ti;
    while (ti * (ti + 1) / 2 > q) --ti;
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = q - ti * (ti + 1) / 2;
  } else {
    // groups of 4 rows of tiles, column by column
    const int grp = q / (4 * nc), in = q - grp * 4 * nc, h = nr - grp * 4 < 4 ? nr - grp * 4 : 4;
    ti = grp * 4 + in % h;
    tj = in / h;
  }
  gchar* ws = (gchar*)it.ws + k * L.bytes();
  const ghalf* P = (const ghalf*)(ws + (PHASE == PHASE_A ? L.x(parity) : PHASE == PHASE_B ? L.a() : L.b()));
  const ghalf* Q = PHASE <= PHASE_B ? P : (const ghalf*)(ws + L.x(parity));
  const int K = PHASE == PHASE_A ? L.cp : L.rp;
  const int qrows = PHASE <= PHASE_B ? L.rp : L.cp;
  const int stage0 = part * chunk, left = K * W / 64 - stage0;
  const int stages = __builtin_amdgcn_readfirstlane(PHASE == PHASE_A && left > chunk ? chunk : left);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
  // Loads: an instruction brings 8 rows of a stage; the first half of them are P's, the others Q's.  (Its rows lie in one
  // of the 64-row parts that operands are padded to: those past the operand are replaced by its tile's first ones, for
  // results that nobody keeps.)
  const char* src[LOADS];
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    const int any = 8 * (l * NW + wave), row = any % TILE, row0 = (any < TILE ? ti : tj) * TILE;
    const int rows = (any < TILE ? L.rp : qrows) - row0;
    const int row1 = row0 + (row < rows ? row : 0);
    if (PHASE >= PHASE_X && any >= TILE)   // 32 columns: 4 instructions
      src[l] = uniform((const char*)Q + (int64_t)(row1 >> 5) * L.rp * (64 * W) + (row >> 3 & 3) * 1024);
    else
      src[l] = uniform((const char*)(any < TILE ? P : Q) + (int64_t)row1 * (64 * W) +
                       (PHASE == PHASE_A ? (int64_t)stage0 * L.rp * 128 : 0));
  }
  // the lane's chunk; in prec 1 a stage's row is two of the operand's 64-byte ones
  const int lrow = lane >> 3, lchunk = (lane & 7) ^ lrow;
  const uint32_t off = lrow * (64 * W) + (W == 1 ? lchunk & 3 : lchunk) * 16;
  const uint32_t offp = off + (W == 1 ? (lchunk >> 2) * L.rp * 64 : 0);
  uint32_t offq = off + (W == 1 ? (lchunk >> 2) * qrows * 64 : 0);
  if (PHASE >= PHASE_X) {
    const int f = W == 1 ? lane >> 5 : (lane >> 4 & 1) | (wave & 1) << 1;   // (an instruction's rows: 8 x its number)
    offq = (lane ^ 2 * f) * 16;
  }
  const auto issue = [&](int s) {
    const uint32_t dst = lds0 + (s % NBUF) * STAGE + wave * 1024;
    const int64_t sp = (int64_t)s * L.rp * 128, sq = PHASE >= PHASE_X ? (int64_t)s * 4096 : (int64_t)s * qrows * 128;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const bool p = 8 * (l * NW + wave) < TILE;
      lds_dma16_s(src[l] + (p ? sp : sq), p ? offp : offq, dst + l * NW * 1024);
    }
  };
  static_assert(LOADS * NW * 8 == 2 * TILE && NW % 2 == 0, "whole instructions");

  floatx4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  // what the epilogue adds to the product: with 64-wide tiles, whose time is waiting, brought along with the operands
  constexpr int G = PHASE == PHASE_LAST ? 4 : 8;   // columns of a thread (8: 1% of all but the large prec 1 products)
  typedef _Float16 halfg __attribute__((ext_vector_type(G)));
  typedef MMS_GLOBAL halfg ghalfg;
  constexpr int OWN = TILE == 64 && PHASE != PHASE_A ? 64 * TILE / G / NT : 0;
  halfg own_hi[OWN + 1], own_lo[OWN + 1];
  // (the last product's results go to rows of the caller's: threads along the row; others as the operands lie: 4 threads
  // for 32 columns, then the next row)
  const auto place = [](int e, int& i, int& j) {
    if (PHASE == PHASE_LAST) { i = e / (TILE / 4); j = e % (TILE / 4) * 4; }
    else { i = e / (32 / G) & 63; j = e / (64 * 32 / G) * 32 + e % (32 / G) * G; }
  };
  const auto own = [&](int i, int j, halfg& hi, halfg& lo) {
    const int64_t d = at<W>(ti * TILE + i, L.rp, tj * TILE + j);
    const ghalf* x = PHASE == PHASE_B ? P : (const ghalf*)(ws + L.x(parity));
    hi = *(const ghalfg*)(x + d);
    if (W == 2) lo = *(const ghalfg*)(x + d + 32);
    else if (PHASE >= PHASE_X) lo = *(const ghalfg*)((const ghalf*)(ws + L.xlo()) + d);
    else lo = halfg(0);
  };
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    int i, j;
    place(threadIdx.x + o * NT, i, j);
    own(i, j, own_hi[o], own_lo[o]);
  }

  // lo is 2^6 times what it stands for, so that it keeps its bits where hi is small; hi lo + lo hi then count 2^-6.  They
  // have a sum of their own, up to tiles of 192: a matrix instruction rounds its sum each time, and these are 2^-11 of
  // hi hi (the renderer's matrices: 0.5 of float32 products' error, 0.7 in one sum).  256-wide tiles have no registers for
  // two sums: there hi, once multiplied by hi, is itself taken 2^-6 times.
  constexpr bool APART = W == 2 && TILE < 256;
  constexpr bool LEAST = W == 2 && TILE == 64;   // a third sum, of lo lo
  floatx4 cross[APART ? FM : 1][APART ? FN : 1], least[LEAST ? FM : 1][LEAST ? FN : 1];
#pragma unroll
  for (int i = 0; i < (APART ? FM : 1); ++i)
#pragma unroll
    for (int j = 0; j < (APART ? FN : 1); ++j) cross[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < (LEAST ? FM : 1); ++i)
#pragma unroll
    for (int j = 0; j < (LEAST ? FN : 1); ++j) least[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  // lo lo too where few singular values leave little to average (3 x 64: 1.1 of float32 products' error on average, 1.6
  // without; from 64 rows it would be 0.5 .. 0.7 for 0.5 .. 0.8, and 7% slower).  Tiles that lack a sum for it go over such
  // a matrix once more for each unit.
  const bool narrow = W == 2 && L.rp == 64;
  const int frow = lane & 15;
  const int fchunk = ((lane >> 4) ^ (lane & 7)) << 4;
  // the lane's place in the two halves of 32 columns of X's rows, and the distance from hi to lo or to the next 32 rows
  int ftr[FN], fnext;
  if (PHASE >= PHASE_X) {
    const int g = lane >> 4, row = g * 8 + (frow >> 2), f = W == 1 ? g & 1 : (lane >> 3 & 1) | (g & 1) << 1;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int u = wn * FN + j;
      ftr[j] = (u >> 1) * 4096 + row * (64 * W) + ((u & 1) ^ f) * 32 + (lane & 3) * 8;
    }
    fnext = W == 1 ? 2048 : 64 - (f >> 1) * 128;
  }
  const auto column = [&](const char* p) {   // 8 rows of a column: two reads of 4
    half8 v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const half4 x = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + h * 256 * W)));
#pragma unroll
      for (int z = 0; z < 4; ++z) v[h * 4 + z] = x[z];
    }
    return v;
  };
  const auto multiply = [&](const half8 (&a)[FM], const half8 (&b)[FN], auto& to) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) to[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[j], to[i][j], 0, 0, 0);
  };
  enum { ALL, LOW_LOW, CROSS, LARGE };   // which products
  const auto sweep = [&](auto which, auto& to, auto& small) {
    constexpr int MODE = decltype(which)::value;
    for (int s = 0; s < NBUF - 1 && s < stages; ++s) issue(s);
    for (int s = 0; s < stages; ++s) {
      // stage s has arrived once only the loads issued after it are outstanding; all waves are then past stage s - 1
      if (s + NBUF - 2 < stages) wait_vm_barrier<(NBUF - 2) * LOADS>();
      else wait_vm_barrier<0>();
      if (s + NBUF - 1 < stages) issue(s + NBUF - 1);
      const char* pa = lds + (s % NBUF) * STAGE + (wm * WM + frow) * 128;
      const char* pq = lds + (s % NBUF) * STAGE + (TILE + (PHASE >= PHASE_X ? 0 : wn * WN + frow)) * 128;
      half8 a0[FM], a1[FM], b0[FN], b1[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) a0[i] = *(const half8*)(pa + i * 2048 + fchunk);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        b0[j] = PHASE >= PHASE_X ? column(pq + ftr[j]) : *(const half8*)(pq + j * 2048 + fchunk);
#pragma unroll
      for (int j = 0; j < FN; ++j)
        b1[j] = PHASE >= PHASE_X ? column(pq + ftr[j] + fnext) : *(const half8*)(pq + j * 2048 + (fchunk ^ 64));
#pragma unroll
      for (int i = 0; i < FM; ++i) a1[i] = *(const half8*)(pa + i * 2048 + (fchunk ^ 64));
      if (MODE == ALL || MODE == LARGE) multiply(a0, b0, to);
      if (W == 1) multiply(a1, b1, to);
      if (W == 2 && !APART && MODE == ALL) {
#pragma unroll
        for (int i = 0; i < FM; ++i) a0[i] *= (_Float16)kUnlow;
#pragma unroll
        for (int j = 0; j < FN; ++j) b0[j] *= (_Float16)kUnlow;
      }
      if (W == 2 && (MODE == ALL || MODE == CROSS)) {
        multiply(a0, b1, small);
        multiply(a1, b0, small);
      }
      if (MODE == LOW_LOW) multiply(a1, b1, small);
      if constexpr (LEAST)
        if (narrow) multiply(a1, b1, least);
    }
  };
  const auto lower = [&](auto& x) {
#pragma unroll
    for (auto& row : x)
#pragma unroll
      for (floatx4& v : row) v *= kUnlow;
  };
  if constexpr (APART) {
    if (!LEAST && narrow) {
      sweep(std::integral_constant<int, LOW_LOW>{}, acc, cross);
      lower(cross);
      __syncthreads();
    }
    sweep(std::integral_constant<int, ALL>{}, acc, cross);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if (LEAST) cross[i][j] += least[LEAST ? i : 0][LEAST ? j : 0] * kUnlow;
        acc[i][j] += cross[i][j] * kUnlow;
      }
  } else if (W == 2 && narrow) {
    sweep(std::integral_constant<int, LOW_LOW>{}, acc, acc);
    lower(acc);
    __syncthreads();
    sweep(std::integral_constant<int, CROSS>{}, acc, acc);
    lower(acc);
    __syncthreads();
    sweep(std::integral_constant<int, LARGE>{}, acc, acc);
  } else {
    sweep(std::integral_constant<int, ALL>{}, acc, acc);
  }
  __syncthreads();
  if (PHASE == PHASE_A && parts > 1) {
    // The sums of a tile in parts: each block leaves its own, the last one to arrive adds them all in their order (which
    // block that is changes nothing) and goes on.  Nobody waits.  Blocks on different XCDs see each other's parts by
    // loads and stores past their L2s (agent scope, 8 bytes each): a fence at that scope in their place writes back all
    // of an L2, for each wave (300 x 4096 in 11 parts: 33 us with fences, 14 so).
    constexpr int EACH = TILE * TILE / 2;
    typedef uint64_t pair2 __attribute__((ext_vector_type(2)));
    uint64_t* to = partial + (int64_t)slot * EACH + threadIdx.x;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const pair2 v = __builtin_bit_cast(pair2, acc[i][j]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          __hip_atomic_store(to + ((i * FN + j) * 2 + h) * NT, v[h], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // they are in memory
    __syncthreads();
    int* arrived = T->arrived + (slot - part * tiles);
    if (threadIdx.x == 0)
      *(int*)lds = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(*(const int*)lds) != parts - 1) return;
    asm volatile("" ::: "memory");
    if (threadIdx.x == 0) *arrived = 0;   // for the next step's launch
    uint64_t* from = partial + (int64_t)(slot - part * tiles) * EACH + threadIdx.x;
    for (int p = 0; p < parts; ++p) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          pair2 v;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            v[h] = __hip_atomic_load(from + ((i * FN + j) * 2 + h) * NT, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          const floatx4 x = __builtin_bit_cast(floatx4, v);
          acc[i][j] = p ? acc[i][j] + x : x;
        }
      from += (int64_t)tiles * EACH;
    }
    __syncthreads();   // lds: the flag was read
  }

  // epilogue: 64 rows at a time through LDS in fp32 (odd row length: columns are read without conflicts too)
  constexpr int LD = TILE + 1;
  float* slab = (float*)lds;
  ghalf* X = (ghalf*)(ws + L.x(parity ^ 1));
  ghalf* Xlo = (ghalf*)(ws + L.xlo());
  ghalf* D = (ghalf*)(ws + (PHASE == PHASE_A ? L.a() : L.b()));
  const bool tall = it.rows > it.cols;
  gchar* out = PHASE == PHASE_LAST ? (gchar*)it.p + k * it.bsp * (bf16 ? 2 : 4) : nullptr;
  const float decay = PHASE == PHASE_LAST && it.m ? (S.hyper ? S.hyper[0] : S.decay) : 0.f;
  const float gain = PHASE == PHASE_LAST ? (it.m ? (S.hyper ? S.hyper[1] : S.neg_lr) * it.scale : 1.f) / S.unit[0] : 0.f;
  // 4 values to the caller's matrix, together where its rows are whole and aligned groups of 4
  const bool quads = PHASE == PHASE_LAST && it.cols % 4 == 0 && it.ldp % 4 == 0 && ((uint64_t)out & (bf16 ? 7 : 15)) == 0;
  const auto put = [&](int row, int col, const float* v) {
    if (row >= it.rows || col >= it.cols) return;
    const int64_t e = (int64_t)row * it.ldp + col;
    float y[4];
    if (quads) {
      MMS_GLOBAL uint64_t* p16 = (MMS_GLOBAL uint64_t*)(out + e * 2);
      MMS_GLOBAL floatx4* p32 = (MMS_GLOBAL floatx4*)(out + e * 4);
      floatx4 old{0.f, 0.f, 0.f, 0.f};
      if (it.m) {
        if (bf16) {
          const uint64_t w = *p16;
#pragma unroll
          for (int z = 0; z < 4; ++z) old[z] = __uint_as_float((uint32_t)(w >> (16 * z)) << 16);
        } else {
          old = *p32;
        }
      }
#pragma unroll
      for (int z = 0; z < 4; ++z) y[z] = it.m ? __builtin_fmaf(old[z], decay, v[z] * gain) : v[z] * gain;
      if (bf16) {
        uint64_t w = 0;
#pragma unroll
        for (int z = 0; z < 4; ++z) w |= (uint64_t)to_bf16(y[z]) << (16 * z);
        *p16 = w;
      } else {
        *p32 = floatx4{y[0], y[1], y[2], y[3]};
      }
      return;
    }
#pragma unroll
    for (int z = 0; z < 4; ++z)
      if (col + z < it.cols)
        store1(out, e + z, bf16, it.m ? __builtin_fmaf(load1(out, e + z, bf16), decay, v[z] * gain) : v[z] * gain);
  };
  const int width = PHASE <= PHASE_B ? L.rp : L.cp;
  for (int s = 0; s < TILE / 64; ++s) {
    if (ti * TILE + s * 64 >= L.rp) break;
    if (s) __syncthreads();
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = wm * WM + i * 16 - s * 64;
      if (row >= 0 && row < 64) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            slab[(row + (lane >> 4) * 4 + e) * LD + wn * WN + j * 16 + frow] = acc[i][j][e] * mul;
      }
    }
    __syncthreads();
    const int i0 = ti * TILE + s * 64, j0 = tj * TILE;
#pragma unroll
    for (int o = 0; o < 64 * TILE / G / NT; ++o) {
      int i, j;
      place(threadIdx.x + o * NT, i, j);
      if (TILE > 64 && j0 + j >= width) continue;
      float v[G];
#pragma unroll
      for (int z = 0; z < G; ++z) v[z] = slab[i * LD + j + z];
      halfg hi, lo;
      if (PHASE != PHASE_A) {
        if (OWN) { hi = own_hi[OWN ? o : 0]; lo = own_lo[OWN ? o : 0]; }
        else own(s * 64 + i, j, hi, lo);
#pragma unroll
        for (int z = 0; z < G; ++z) {
          const float y = __builtin_fmaf((float)lo[z], kUnlow, (float)hi[z]);
          v[z] = PHASE == PHASE_B ? __builtin_fmaf(cb, y, cc * v[z]) : __builtin_fmaf(ca, y, v[z]);
        }
      }
      if (PHASE == PHASE_B || PHASE == PHASE_LAST) {
#pragma unroll
        for (int z = 0; z < G; ++z) slab[i * LD + j + z] = v[z];
      }
      if (PHASE == PHASE_LAST) {
        if (!tall) put(i0 + i, j0 + j, v);
      } else {
        split_n<G>(v, (_Float16*)&hi, (_Float16*)&lo);
        const int64_t d = at<W>(i0 + i, L.rp, j0 + j);
        ghalf* to = PHASE == PHASE_X ? X : D;
        *(ghalfg*)(to + d) = hi;
        if (W == 2) *(ghalfg*)(to + d + 32) = lo;
        else if (PHASE == PHASE_X) *(ghalfg*)(Xlo + d) = lo;
      }
    }
    // the other order: the mirrored triangle, or a tall result
    if (PHASE == PHASE_X || (PHASE <= PHASE_B && ti == tj)) continue;
    if (PHASE == PHASE_LAST && !tall) continue;
    __syncthreads();
    for (int e = threadIdx.x; e < 64 * TILE / 8; e += NT) {
      // operands: 4 threads for a row's 32 columns, then the next row; a result: 8 threads along the caller's row
      const int f = PHASE == PHASE_LAST ? e >> 3 : e >> 2, j = f % TILE;
      const int i = PHASE == PHASE_LAST ? (e & 7) * 8 : f / TILE * 32 + (e & 3) * 8;
      if (TILE > 64 && j0 + j >= width) continue;
      float v[8];
#pragma unroll
      for (int z = 0; z < 8; ++z) v[z] = slab[(i + z) * LD + j];
      if (PHASE == PHASE_LAST) {
        put(j0 + j, i0 + i, v);
        put(j0 + j, i0 + i + 4, v + 4);
      } else {
        half8 hi, lo;
        split_n<8>(v, (_Float16*)&hi, (_Float16*)&lo);
        ghalf* d = D + at<W>(j0 + j, width, i0 + i);
        *(ghalf8*)d = hi;
        if (W == 2) *(ghalf8*)(d + 32) = lo;
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
// Operands of hi and lo: prec 0, and matrices whose results have too few entries for the roundings to average out.
int width_of(int64_t rows, int64_t cols, int prec) { return prec == 0 || rows <= 128 || cols <= 128 ? 2 : 1; }

// The launches of the matrices that share one table
struct NsPlan {
  int n, w;                            // matrices (or stacks), operands' width
  int64_t norm, pack, a, b, x;         // blocks
  NsTiles tiles;
  int64_t partial;                     // bytes of A's parts
};

// The tile of a launch whose item i has `count(i, t)` tiles of `stages(i)` stages: the one whose last block should end
// first.  Blocks start with the longest; a CU is busy for cost x (stages + 8) of each of its tiles (8: the epilogue), so
// the end is neither before the n-th longest block had its turn on one of 256 CUs nor before the average CU is through.
// Costs in us, from launches that fill the card: 64-wide tiles are bound by LDS reads, 128 by those and by products,
// 192 and 256 by power (the clock falls to 1.6 GHz under 256-wide tiles, 1.2 PFLOP/s of fp16).  4096 x 4096, prec 1: A
// 158, 110, 87, 108 us with 64, 128, 192, 256-wide tiles (253 of the 192-wide ones: one for each CU), X 232, 163, 194,
// 138; six of 701 x 1100, prec 0: A 20, 28, 46, 68 us, X 32, 33, 40, 54.
// With `chunk`, tiles may be summed in parts of that many stages: as few parts as fill the card with one round of
// blocks, and no more than the square root of the stages (a stage takes about as long as the adding of a part), where
// that beats whole sums.  Parts cost 2 us, for their way through memory, and 0.3 for each that the last block adds.  Only
// tiles up to 128 are split: with 256-wide ones a whole call was 9 .. 14% slower for it (2 x 501 x 991 with 2033 x 7973
// prec 0: 2335 us, 2033 with the choice below), with 192-wide ones 7% faster to 4% slower.
// prec 0: 64 x 4096 (128 stages) 38 us whole, 13 in 11 parts; 100 x 20000 (626) 177, 22 in 25 parts (29 in 53);
// 300 x 4096 with 60 x 2000 and 1000 x 1000 40, 17.
constexpr int kTiles[4] = {256, 192, 128, 64}, kPerCu[4] = {1, 1, 2, 3};
constexpr float kGramCost[2][4] = {{1.90f, 1.22f, 0.55f, 0.23f}, {2.25f, 1.40f, 0.73f, 0.26f}};
constexpr float kFullCost[2][4] = {{1.90f, 1.38f, 0.60f, 0.22f}, {2.00f, 1.38f, 0.62f, 0.21f}};
// Estimates that come to the same go to the wider tile and to whole sums, not to a float's last bit: another tile has to
// gain 0.1%, a split 5%, and 20% with 128-wide tiles of single fp16 operands, whose parts are the most traffic beside
// their products (prec 1, a whole call, whole sums and split: 8 x 1024 x 4096 978 and 1050 us, 8 x 1071 x 8055 2216 and
// 2310, 4 x 671 x 13842 1088 and 1043).
constexpr float kTie = 0.999f, kSplit = 0.95f, kWideSplit = 0.8f;
constexpr int kMinChunk = 12;
template <typename Count, typename Stages>
int choose_tile(int n, int w, const float (&cost)[4], const Count& count, const Stages& stages, int* chunk) {
  int best = 64;
  float least = 1e30f;
  for (int k = 0; k < 4; ++k) {
    int64_t total = 0;
    int longest = 0;
    for (int whole = 1; whole >= (chunk && kTiles[k] <= 128 ? 0 : 1); --whole) {
      int len = 1 << 30;
      if (!whole) {
        // the longest sum in equal parts, the others in parts of the same length
        const int64_t fill = (total + 256 * kPerCu[k] - 1) / (256 * kPerCu[k]);
        const int least_len = std::max(kMinChunk, (int)sqrtf((float)longest));
        const int l = (int)std::min<int64_t>(std::max<int64_t>(fill, least_len), longest);
        const int parts = (longest + l - 1) / l;
        if (parts < 2) break;
        len = (longest + parts - 1) / parts;
      }
      int64_t before = 0;
      float sum = 0.f, end = 0.f;
      for (int i = 0; i < n; ++i) {
        const int s = stages(i), parts = (int)(((int64_t)s + len - 1) / len);
        const int64_t c = count(i, kTiles[k]) * parts;
        const float each = cost[k] * (8 + std::min(s, len)) + (parts > 1 ? 2.f + 0.3f * parts * (kTiles[k] / 64) * (kTiles[k] / 64) : 0.f);
        before += c;
        sum += each * c;
        end = fmaxf(end, each * ((before + 255) / 256));
        total += whole ? c * s : 0;
        longest = s > longest ? s : longest;
      }
      end = fmaxf(end, sum / 256);
      if (!whole && before > kMaxParts) continue;
      if (end < least * (whole ? kTie : w == 1 && kTiles[k] > 64 ? kWideSplit : kSplit)) {
        least = end;
        best = kTiles[k];
        if (chunk) *chunk = len;
      }
    }
  }
  return best;
}

int ns_check(const char* fn, int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec) {
  MMS_REQUIRE(n >= 0 && n <= kMaxMatrices, fn, "0 to 4096 matrices");
  MMS_REQUIRE(n == 0 || (batch && rows && cols), fn, "null size table");
  MMS_REQUIRE(prec == 0 || prec == 1, fn, "prec 0 (split fp16) or 1 (fp16)");
  for (int i = 0; i < n; ++i)
    MMS_REQUIRE(batch[i] >= 0 && rows[i] >= 0 && cols[i] >= 0 && batch[i] <= (1 << 20) && rows[i] <= (1 << 20) &&
                    cols[i] <= (1 << 20) && batch[i] * ((rows[i] + 255) / 256) * ((cols[i] + 255) / 256) * 16 <= kMaxBlocks &&
                    batch[i] * ((rows[i] * cols[i] + kNormElems - 1) / kNormElems) <= kMaxBlocks,
                fn, "matrix sizes up to 2^20 a side and 2^23 64 x 64 tiles a stack");
  return 0;
}

// The plan of the next matrices of `order` that one table holds: the first ones, as long as they have one width
NsPlan plan_group(const int* order, int live, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec) {
  NsPlan P{};
  P.w = width_of(rows[order[0]], cols[order[0]], prec);
  const auto layout = [&](int i) { return NsLayout((int)rows[order[i]], (int)cols[order[i]], P.w); };
  for (; P.n < live && P.n < kNsItems; ++P.n) {
    const int i = order[P.n];
    if (width_of(rows[i], cols[i], prec) != P.w) break;
    const int64_t norm = batch[i] * norm_blocks(rows[i], cols[i]), pack = batch[i] * pack_blocks(layout(P.n));
    if (P.n && (P.norm + norm > kMaxBlocks || P.pack + pack > kMaxBlocks)) break;
    P.norm += norm;
    P.pack += pack;
  }
  const auto gram = [&](int i, int t) { return gram_blocks(layout(i), t) * batch[order[i]]; };
  const auto full = [&](int i, int t) { return full_blocks(layout(i), t) * batch[order[i]]; };
  const auto along = [&](int i) { return layout(i).cp * P.w / 64; };
  const auto across = [&](int i) { return layout(i).rp * P.w / 64; };
  P.tiles.a = choose_tile(P.n, P.w, kGramCost[P.w - 1], gram, along, &P.tiles.chunk);
  P.tiles.b = choose_tile(P.n, P.w, kGramCost[P.w - 1], gram, across, nullptr);
  P.tiles.x = choose_tile(P.n, P.w, kFullCost[P.w - 1], full, across, nullptr);
  bool split = false;
  for (int i = 0; i < P.n; ++i) {
    const int parts = gram_parts(layout(i), P.tiles.chunk);
    split = split || parts > 1;
    P.a += gram(i, P.tiles.a) * parts;
    P.b += gram(i, P.tiles.b);
    P.x += full(i, P.tiles.x);
  }
  P.partial = split ? P.a * P.tiles.a * P.tiles.a * (int64_t)sizeof(float) : 0;
  return P;
}

// The matrices that are not empty, by width, largest first: their blocks are started first
int sort_matrices(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec, int* order) {
  int live = 0;
  for (int i = 0; i < n; ++i)
    if (batch[i] * rows[i] * cols[i] > 0) order[live++] = i;
  std::sort(order, order + live, [&](int i, int j) {
    const int v = width_of(rows[i], cols[i], prec), w = width_of(rows[j], cols[j], prec);
    const int64_t x = rows[i] + cols[i], y = rows[j] + cols[j];
    return v != w ? v < w : x != y ? x > y : i < j;
  });
  return live;
}

// The workspace: A's parts, which the groups use in turn (`partial` bytes), then each group's table and operands.
int64_t workspace_of(const int* order, int live, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec,
                     NsPlan& first, int64_t& partial) {
  int64_t bytes = 0;
  partial = 0;
  for (int at = 0; at < live;) {
    const NsPlan P = plan_group(order + at, live - at, batch, rows, cols, prec);
    if (at == 0) first = P;
    bytes += kTableBytes;
    for (int i = 0; i < P.n; ++i, ++at)
      bytes += batch[order[at]] * NsLayout((int)rows[order[at]], (int)cols[order[at]], P.w).bytes();
    partial = P.partial > partial ? P.partial : partial;
  }
  return bytes + partial;
}

template <int W, int PHASE>
void launch_product(int tile, NsTable* T, int64_t blocks, const NsStep& S, float a, float b, float c, int parity,
                    int bf16, int chunk, uint64_t* partial, hipStream_t s) {
  // a sum's factor, to hold A, A A in A's unit, B X in X's; then B's unit for A's
  const float x = S.unit[0], aa = S.unit[1], bb = S.unit[2];
  const float mul = PHASE == PHASE_A ? aa / (x * x) : 1.f / (PHASE == PHASE_B ? aa : bb);
  b *= bb / aa;
  c *= bb / aa;
  const dim3 grid((unsigned)blocks);
#define NS_LAUNCH(TILE, WM, WN, NBUF)                                                                            \
  hipLaunchKernelGGL((ns_product_kernel<TILE, WM, WN, NBUF, W, PHASE>), grid, dim3((TILE / WM) * (TILE / WN) * 64), 0, \
                     s, T, S, mul, a, b, c, parity, bf16, chunk, partial)
  // 16 waves a CU where registers and LDS allow it: 8-wave blocks of 128 two at a time (X of four 2048 x 2048 and two
  // 2048 x 5632 in prec 0: 2% faster than 4 waves), 16 of 64 x 64 rather than 8 of 128 x 64 for 256 (5%), 4-wave blocks
  // of 64 three at a time
  if (tile == 64) NS_LAUNCH(64, 32, 32, 3);
  else if (tile == 128) NS_LAUNCH(128, 64, 32, 2);
  else if (tile == 192) NS_LAUNCH(192, 64, 48, 3);
  else NS_LAUNCH(256, 64, 64, 2);
#undef NS_LAUNCH
}

template <int W>
void launch_group(const NsPlan& P, const NsArgs& A, NsTable* T, const NsStep& S, int steps, float a, float b, float c,
                  int bf16, uint64_t* partial, hipStream_t s) {
  hipLaunchKernelGGL(muon_momentum_kernel, dim3((unsigned)P.norm), dim3(256), 0, s, A, S, bf16, W, P.tiles, T);
  hipLaunchKernelGGL((ns_pack_kernel<W>), dim3((unsigned)P.pack), dim3(256), 0, s, T, S, bf16);
  for (int i = 0; i < steps; ++i) {
    launch_product<W, PHASE_A>(P.tiles.a, T, P.a, S, a, b, c, i & 1, bf16, P.tiles.chunk, partial, s);
    launch_product<W, PHASE_B>(P.tiles.b, T, P.b, S, a, b, c, i & 1, bf16, 0, nullptr, s);
    if (i + 1 < steps) launch_product<W, PHASE_X>(P.tiles.x, T, P.x, S, a, b, c, i & 1, bf16, 0, nullptr, s);
    else launch_product<W, PHASE_LAST>(P.tiles.x, T, P.x, S, a, b, c, i & 1, bf16, 0, nullptr, s);
  }
}

// The operands' units: the largest powers of two, up to 2^15, with which no entry can pass fp16's range.  Entries are at
// most the largest singular value, which starts at 1 or less; p(s) = a s + b s^3 + c s^5 takes [0, m] onto [0, max |p|]
// (and beyond zero), B has b t + c t^2 for t in [0, m^2].  False: some matrix's iterates leave the range.
bool ns_units(int steps, double a, double b, double c, float (&unit)[3]) {
  constexpr double margin = 1.01;   // roundings: a singular value may be a little larger than exactly computed
  double m = margin, x = 0.0, poly = 0.0;
  for (int i = 0; i < steps; ++i) {
    x = std::max(x, m);
    const double t = m * m;
    double next = 0.0;
    const auto see_p = [&](double s) { next = std::max(next, fabs(s * (a + s * s * (b + s * s * c)))); };
    const auto see_b = [&](double u) { poly = std::max(poly, fabs(u * (b + c * u))); };
    see_p(m);
    see_b(t);
    if (c != 0.0) {
      const double d = 9.0 * b * b - 20.0 * a * c;
      for (int sign = -1; sign <= 1 && d >= 0.0; sign += 2) {   // p' = a + 3 b s^2 + 5 c s^4
        const double u = (-3.0 * b + sign * sqrt(d)) / (10.0 * c);
        if (u > 0.0 && u < t) see_p(sqrt(u));
      }
      if (const double u = -b / (2.0 * c); u > 0.0 && u < t) see_b(u);
    } else if (b != 0.0) {
      if (const double u = -a / (3.0 * b); u > 0.0 && u < t) see_p(sqrt(u));
    }
    if (!(next < 1e30)) { m = next; if (i + 1 < steps) return false; break; }
    m = next * margin;
  }
  const double largest[3] = {x, x * x, poly * margin};
  for (int i = 0; i < 3; ++i) {
    if (!(largest[i] <= kHalfMax)) return false;
    int e = 15;
    while (e > 0 && ldexp(largest[i], e) > kHalfMax) --e;
    unit[i] = (float)(1 << e);
  }
  return true;
}

// ---- what a call writes may not be read or written by another of its matrices: their blocks run together ------------
// Rows of `width` bytes, `ld` apart, in matrices `bs` apart, ascending and apart (of what is written: checked before).
struct Rows {
  uintptr_t lo, hi;      // first byte, past the last
  int64_t width, ld, bs, rows, batch;
  int matrix, kind;      // 0 gradients, 1 weights or results, 2 momenta
};

Rows rows_of(const void* p, int64_t es, int64_t rows, int64_t cols, int64_t ld, int64_t batch, int64_t bs, int matrix,
             int kind) {
  Rows r{(uintptr_t)p, 0, cols * es, rows > 1 ? ld * es : cols * es, batch > 1 ? bs * es : 0, rows, batch, matrix, kind};
  r.hi = r.lo + (uintptr_t)((batch - 1) * r.bs + (rows - 1) * r.ld + r.width);
  return r;
}

// does any row of `b` reach into [x, x + width)?
bool reaches(const Rows& b, uintptr_t x, int64_t width) {
  const int64_t y = (int64_t)(x - b.lo) + width - 1;   // the last byte, from b's first
  if (y < 0) return false;
  const int64_t k = b.batch > 1 ? std::min(y / b.bs, b.batch - 1) : 0, r = std::min((y - k * b.bs) / b.ld, b.rows - 1);
  return k * b.bs + r * b.ld + b.width > y - width + 1;   // the last row that begins by then
}

bool overlap(const Rows& a, const Rows& b) {
  if (a.hi <= b.lo || b.hi <= a.lo) return false;
  const auto apart = [](const Rows& r) { return r.batch == 1 || r.bs >= (r.rows - 1) * r.ld + r.width; };
  if (!apart(a) || !apart(b)) return true;   // a repeated gradient: not looked at row by row
  const Rows &few = a.rows * a.batch <= b.rows * b.batch ? a : b, &many = &few == &a ? b : a;
  // columns of one buffer, side by side
  if (a.ld == b.ld && a.bs % a.ld == 0 && b.bs % a.ld == 0) {
    const int64_t from = (int64_t)(many.lo - few.lo) % a.ld, d = from < 0 ? from + a.ld : from;
    if (d >= few.width && d + many.width <= a.ld) return false;
  }
  for (int64_t k = 0; k < few.batch; ++k)
    for (int64_t r = 0; r < few.rows; ++r)
      if (reaches(many, few.lo + (uintptr_t)(k * few.bs + r * few.ld), few.width)) return true;
  return false;
}

// 0, or 1 if one of the call's matrices writes what another reads or writes, or its own momentum and weights or gradient
// are not apart (a weight may lie where its own gradient does: that is read before).
int conflict(Rows* all, int n) {
  std::sort(all, all + n, [](const Rows& a, const Rows& b) { return a.lo < b.lo; });
  uintptr_t reach = 0;   // of the rows before
  for (int i = 0; i < n; ++i) {
    if (all[i].lo < reach)
      for (int j = 0; j < i; ++j) {
        const Rows &a = all[i], &b = all[j];
        if (a.kind + b.kind == 0 || (a.matrix == b.matrix && a.kind + b.kind == 1)) continue;
        if (overlap(a, b)) return 1;
      }
    reach = std::max(reach, all[i].hi);
  }
  return 0;
}

int ns_run(const char* fn, int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, void* const* p,
           const int64_t* ldp, const int64_t* bsp, const void* const* g, const int64_t* ldg, const int64_t* bsg,
           float* const* m, const float* scale, int bf16, int prec, int steps, float a, float b, float c,
           NsStep S, void* ws, int64_t ws_bytes, void* stream) {
  MMS_REQUIRE(steps >= 1 && steps <= 64, fn, "1 to 64 steps");
  MMS_REQUIRE(S.eps > 0.0, fn, "eps must be positive");
  MMS_REQUIRE(ns_units(steps, a, b, c, S.unit), fn,
              "coefficients with which X, X X^T or b A + c A A can pass 60000 in fewer steps than these");
  MMS_REQUIRE(n == 0 || (p && ldp && bsp && g && ldg && bsg), fn, "null pointer table");
  const int rc = ns_check(fn, n, batch, rows, cols, prec);
  if (rc) return rc;
  static thread_local int order[kMaxMatrices];
  const int live = sort_matrices(n, batch, rows, cols, prec, order);
  NsPlan P{};
  int64_t parts = 0;
  const int64_t need = workspace_of(order, live, batch, rows, cols, prec, P, parts);
  for (int i = 0; i < n; ++i) {
    if (batch[i] * rows[i] * cols[i] == 0) continue;
    MMS_REQUIRE(p[i] && g[i], fn, "null matrix");
    MMS_REQUIRE(ldp[i] >= cols[i] && ldg[i] >= cols[i] && ldp[i] < (1LL << 31) && ldg[i] < (1LL << 31), fn,
                "leading dimensions must hold a row");
    MMS_REQUIRE(bsp[i] >= 0 && bsg[i] >= 0 && (batch[i] == 1 || bsp[i] >= rows[i] * ldp[i] - (ldp[i] - cols[i])), fn,
                "stacked matrices must not overlap");
  }
  const char* small = "workspace too small (mms_muon_workspace) or not 256-byte aligned";
  MMS_REQUIRE(need == 0 || ws, fn, small);
  if (live) {
    Rows* all = new (std::nothrow) Rows[3 * live];
    MMS_REQUIRE(all != nullptr, fn, "out of host memory");
    int count = 0;
    const int64_t es = bf16 ? 2 : 4;
    for (int k = 0; k < live; ++k) {
      const int i = order[k];
      all[count++] = rows_of(g[i], es, rows[i], cols[i], ldg[i], batch[i], bsg[i], i, 0);
      all[count++] = rows_of(p[i], es, rows[i], cols[i], ldp[i], batch[i], bsp[i], i, 1);
      if (m) all[count++] = rows_of(m[i], 4, rows[i], cols[i], cols[i], batch[i], rows[i] * cols[i], i, 2);
    }
    const int bad = conflict(all, count);
    delete[] all;
    MMS_REQUIRE(bad == 0, fn, "matrices that are written must not overlap others of the call");
  }
  MMS_REQUIRE(need == 0 || (ws_bytes >= need && ((uintptr_t)ws & 255) == 0), fn, small);
  hipStream_t s = mms::as_stream(stream);
  uint64_t* partial = (uint64_t*)ws;
  char* next = (char*)ws + parts;
  for (int at = 0; at < live;) {
    if (at) P = plan_group(order + at, live - at, batch, rows, cols, prec);
    NsTable* T = (NsTable*)next;
    next += kTableBytes;
    NsArgs A{};
    A.n = P.n;
    int64_t norm = 0;
    for (int k = 0; k < P.n; ++k, ++at) {
      const int i = order[at];
      A.it[k] = NsItem{g[i], m ? m[i] : nullptr, p[i], next, bsg[i], bsp[i], (int)ldg[i], (int)ldp[i], (int)rows[i],
                       (int)cols[i], (int)batch[i], scale ? scale[i] : 1.f};
      A.blk0[k] = (int)norm;
      next += batch[i] * NsLayout((int)rows[i], (int)cols[i], P.w).bytes();
      norm += batch[i] * norm_blocks(rows[i], cols[i]);
    }
    A.blk0[P.n] = (int)norm;
    if (P.w == 1) launch_group<1>(P, A, T, S, steps, a, b, c, bf16, partial, s);
    else launch_group<2>(P, A, T, S, steps, a, b, c, bf16, partial, s);
    const int e = mms::check_launch(fn);
    if (e) return e;
  }
  return 0;
}

}  // namespace

MMS_EXPORT int mms_muon_workspace(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec,
                                  int64_t* bytes) {
  const char* fn = "mms_muon_workspace";
  MMS_REQUIRE(bytes != nullptr, fn, "null output");
  const int rc = ns_check(fn, n, batch, rows, cols, prec);
  if (rc) return rc;
  static thread_local int order[kMaxMatrices];
  NsPlan first;
  int64_t partial;
  *bytes = workspace_of(order, sort_matrices(n, batch, rows, cols, prec, order), batch, rows, cols, prec, first, partial);
  return 0;
}

MMS_EXPORT int mms_muon_plan(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec, int max,
                             int64_t* plan, int64_t* tables) {
  const char* fn = "mms_muon_plan";
  MMS_REQUIRE(tables != nullptr && (plan != nullptr || max <= 0), fn, "null output");
  const int rc = ns_check(fn, n, batch, rows, cols, prec);
  if (rc) return rc;
  static thread_local int order[kMaxMatrices];
  const int live = sort_matrices(n, batch, rows, cols, prec, order);
  *tables = 0;
  for (int at = 0; at < live; ++*tables) {
    const NsPlan P = plan_group(order + at, live - at, batch, rows, cols, prec);
    if (*tables < max) {
      int64_t* out = plan + 6 * *tables;
      out[0] = P.n;
      out[1] = P.w;
      out[2] = P.tiles.a;
      out[3] = P.partial ? P.tiles.chunk : 0;
      out[4] = P.tiles.b;
      out[5] = P.tiles.x;
    }
    at += P.n;
  }
  return 0;
}

MMS_EXPORT int mms_newton_schulz(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols,
                                 const void* const* g, const int64_t* ldg, const int64_t* bsg, void* const* out,
                                 const int64_t* ldo, const int64_t* bso, int bf16, int prec, int steps, float a, float b,
                                 float c, double eps, void* ws, int64_t ws_bytes, void* stream) {
  NsStep S{};
  S.eps = eps;
  return ns_run("mms_newton_schulz", n, batch, rows, cols, out, ldo, bso, g, ldg, bsg, nullptr, nullptr, bf16, prec,
                steps, a, b, c, S, ws, ws_bytes, stream);
}

MMS_EXPORT int mms_muon_step(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, void* const* p,
                             const int64_t* ldp, const int64_t* bsp, const void* const* g, const int64_t* ldg,
                             const int64_t* bsg, float* const* m, const float* scale, int bf16, int prec, int steps,
                             float a, float b, float c, double eps, double momentum, int nesterov, const float* sumsq,
                             float max_norm, const float* hyper, float decay, float neg_lr, void* ws, int64_t ws_bytes,
                             void* stream) {
  const char* fn = "mms_muon_step";
  MMS_REQUIRE(n <= 0 || (m && scale), fn, "null momentum or scale table");
  MMS_REQUIRE(momentum >= 0.0 && momentum < 1.0, fn, "momentum must be in [0, 1)");
  for (int i = 0; i < n; ++i) MMS_REQUIRE(m[i] || !rows || !cols || !batch || batch[i] * rows[i] * cols[i] == 0, fn, "null momentum");
  const NsStep S{(float)momentum, (float)(1.0 - momentum), nesterov, sumsq, max_norm, hyper, decay, neg_lr, eps, {}};
  return ns_run(fn, n, batch, rows, cols, p, ldp, bsp, g, ldg, bsg, m, scale, bf16, prec, steps, a, b, c, S, ws,
                ws_bytes, stream);
}
