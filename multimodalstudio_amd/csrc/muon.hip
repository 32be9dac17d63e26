// Muon's update of weight matrices: the momentum, its orthogonalisation by Newton-Schulz products, the weights.
//
//   m <- m + (1 - mu)(g - m),  u = g + mu (m - g) (Nesterov) or m             (g clipped by its group's norm)
//   X = u / max(|u|_F, eps)                                                     on the side with fewer rows: r <= c
//   X <- a X + (b A + c A A) X,  A = X X^T                                      `steps` times
//   p <- decay p - lr scale X
//
// Three products a step, all "rows times rows" (k contiguous in both operands): A = X X^T reads the rows of X; A A the
// rows of A, which is symmetric; the last one the rows of B = b A + c A A and of X^T, so every product's epilogue
// writes the operand layouts that the next ones read (X and X^T, or both triangles) and the loop needs no transposing
// load.  A and B are symmetric: only tiles on or below the diagonal are computed, the others are written as mirrors --
// 3 r^2 c + r^3 multiply-adds a step in place of 4 r^2 c + 2 r^3.
//
// Precision.  Operands are fp16 with |X| <= 1.2 held as 2^10 X (entries from 2^-24 of the largest possible keep their
// bits); fp32 accumulators.
//   prec 0  x = hi + lo, both fp16 (22 bits); a product is hi hi + hi lo + lo hi: as near the definition as fp32
//           products, at a third of the fp16 matrix rate (fp32 MFMA: a sixteenth).  bf16 pairs hold 16 bits only,
//           which the map's slope (up to a^5 = 485 for small singular values) takes to 3e-5 .. 2e-4.
//   prec 1  one fp16 product.  X itself keeps hi + lo and a X is added from those in fp32: rounding only enters
//           through (b A + c A A) X, so the result is 0.9e-3 .. 1.4e-3 off, under bf16's own 1.7e-3 (X rounded to fp16
//           between steps: up to 1.2e-2 where a few directions are far stronger than the rest).  Small matrices
//           (64-wide tiles) run prec 0 all the same: they wait for launches and loads, not for products, and with few
//           entries to average over, single products are up to 3.8e-3 off.
//
// Every matrix of a call takes part in the same 2 + 3 steps launches; a block finds its matrix and tile by blockIdx.
// Padded rows and columns (to the tile) are zeros in every operand, so the product loop has no bounds checks.
#include "common.h"
#include "chain_common.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kNsItems = 48;             // matrices (or stacks of them) per launch: the argument struct stays < 4 KB
constexpr float kScale = 1024.f;         // fp16 operands hold 2^10 times their value
constexpr float kDescale = 1.f / 1024.f; // a product of two of them, back to 2^10 times its value
constexpr int kNormBlocks = 1024;        // blocks per matrix that sum squares, at most
constexpr int kNormElems = 8192;         // elements per such block, at least

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

struct NsStep {
  float momentum, rest;     // mu and 1 - mu, each rounded once (1 - 0.95f is 2e-7 off)
  int nesterov;
  const float* sumsq;       // of the whole gradient, or null: no clipping
  float max_norm;
  const float* hyper;       // device [decay, -lr], or null: the two values
  float decay, neg_lr;
  double eps;
};

// The workspace of one matrix: norm partials, then the fp16 operands.  W: 2 with hi and lo (32 of each in turn along
// k, so that a 128-byte line holds both), 1 with hi only.
struct NsLayout {
  int rp, cp, w;
  __host__ __device__ NsLayout(int rows, int cols, int tile, int w_) : w(w_) {
    const int r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
    rp = (r + tile - 1) / tile * tile;
    cp = (c + tile - 1) / tile * tile;
  }
  __host__ __device__ int64_t x() const { return kNormBlocks * (int64_t)sizeof(double); }
  __host__ __device__ int64_t xt(int i) const { return x() + (int64_t)rp * cp * w * 2 * (1 + i); }
  __host__ __device__ int64_t a() const { return x() + (int64_t)rp * cp * w * 6; }
  __host__ __device__ int64_t b() const { return a() + (int64_t)rp * rp * w * 2; }
  __host__ __device__ int64_t xlo() const { return b() + (int64_t)rp * rp * w * 2; }
  __host__ __device__ int64_t bytes() const { return xlo() + (w == 1 ? (int64_t)rp * cp * 2 : 0); }
};

__device__ __forceinline__ int find_item(const NsArgs& A, int blk) {
  int lo = 0, hi = A.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (A.blk0[mid] <= blk) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float load1(const void* p, int64_t i, bool bf16) {
  if (bf16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return ((const float*)p)[i];
}
__device__ __forceinline__ uint16_t to_bf16(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ void store1(void* p, int64_t i, bool bf16, float v) {
  if (bf16) ((uint16_t*)p)[i] = to_bf16(v);
  else ((float*)p)[i] = v;
}

__device__ __forceinline__ float clip_of(const NsStep& s) {
  if (!s.sumsq) return 1.f;
  const float c = s.max_norm / (sqrtf(s.sumsq[0]) + 1e-6f);
  return c < 1.f ? c : 1.f;
}

// ---- momentum and the sum of squares ----------------------------------------------------------------------------
// Reads g and m, writes m (12 bytes an element in fp32), and leaves each block's sum of u^2, in double: gradients of
// 1e-25 or 1e25 keep their norm.  u is not stored: the next launch forms it again from the g and m it has to read.
__global__ __launch_bounds__(256) void muon_momentum_kernel(NsArgs A, NsStep S, int bf16, int tile, int w) {
  __shared__ double red[4];
  const int ii = find_item(A, blockIdx.x);
  const NsItem it = A.it[ii];
  const NsLayout L(it.rows, it.cols, tile, w);
  const int per = (A.blk0[ii + 1] - A.blk0[ii]) / it.batch;
  const int k = (blockIdx.x - A.blk0[ii]) / per, b = (blockIdx.x - A.blk0[ii]) % per;
  const int64_t n = (int64_t)it.rows * it.cols;
  const char* g = (const char*)it.g + k * it.bsg * (bf16 ? 2 : 4);
  float* m = it.m ? it.m + k * n : nullptr;
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
  if (dense && n % 4 == 0 && ((uintptr_t)g & (bf16 ? 7 : 15)) == 0 && ((uintptr_t)m & 15) == 0) {
    for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < n / 4; i += step) {
      float gi[4];
      if (bf16) {
        const uint2 q = ((const uint2*)g)[i];
        gi[0] = __uint_as_float(q.x << 16); gi[1] = __uint_as_float(q.x & 0xffff0000u);
        gi[2] = __uint_as_float(q.y << 16); gi[3] = __uint_as_float(q.y & 0xffff0000u);
      } else {
        const float4 q = ((const float4*)g)[i];
        gi[0] = q.x; gi[1] = q.y; gi[2] = q.z; gi[3] = q.w;
      }
      float4 mi = m ? ((const float4*)m)[i] : float4{0.f, 0.f, 0.f, 0.f};
      one(4 * i, gi[0], mi.x); one(4 * i + 1, gi[1], mi.y); one(4 * i + 2, gi[2], mi.z); one(4 * i + 3, gi[3], mi.w);
      if (m) ((float4*)m)[i] = mi;
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

// position of (row, k) in an operand of K columns: with hi and lo, 32 of each in turn
template <int W>
__device__ __forceinline__ int64_t at(int64_t row, int64_t K, int k) {
  return W == 1 ? row * K + k : row * K * 2 + (k >> 5) * 64 + (k & 31);
}

template <int N>
__device__ __forceinline__ void split_n(const float* v, _Float16* hi, _Float16* lo) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    hi[q] = (_Float16)v[q];
    lo[q] = (_Float16)(v[q] - (float)hi[q]);
  }
}

// ---- X and X^T of u / |u| -----------------------------------------------------------------------------------------
// One 64 x 64 tile of u per block through LDS, written in both orders; the rows and columns of the padding as zeros.
template <int W>
__global__ __launch_bounds__(256) void ns_pack_kernel(NsArgs A, NsStep S, int bf16, int tile) {
  __shared__ float t[64][65];
  __shared__ double red[4];
  const int ii = find_item(A, blockIdx.x);
  const NsItem it = A.it[ii];
  const NsLayout L(it.rows, it.cols, tile, W);
  const bool tall = it.rows > it.cols;
  const int tr = (tall ? L.cp : L.rp) / 64, tc = (tall ? L.rp : L.cp) / 64;
  const int q = blockIdx.x - A.blk0[ii];
  const int k = q / (tr * tc), i0 = (q / tc) % tr * 64, j0 = q % tc * 64;
  char* ws = it.ws + k * L.bytes();
  const int64_t n = (int64_t)it.rows * it.cols;
  // |u|: the partial sums in a fixed order
  const int64_t nb64 = (n + kNormElems - 1) / kNormElems;
  const int nb = nb64 < 1 ? 1 : nb64 > kNormBlocks ? kNormBlocks : (int)nb64;
  double sum = 0.0;
  for (int i = threadIdx.x; i < nb; i += 256) sum += ((const double*)ws)[i];
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  norm = norm < S.eps ? S.eps : norm;
  const double inv = (double)kScale / norm;

  const char* g = (const char*)it.g + k * it.bsg * (bf16 ? 2 : 4);
  const float* m = it.m ? it.m + k * n : nullptr;
  const float clip = clip_of(S), mu = S.momentum;
  for (int e = threadIdx.x; e < 64 * 64; e += 256) {
    const int i = i0 + (e >> 6), j = j0 + (e & 63);
    float u = 0.f;
    if (i < it.rows && j < it.cols) {
      const float gi = load1(g, (int64_t)i * it.ldg + j, bf16) * clip;
      u = gi;
      if (m) {
        const float mi = m[(int64_t)i * it.cols + j];
        u = S.nesterov ? __builtin_fmaf(mu, mi - gi, gi) : mi;
      }
      u = (float)(u * inv);
    }
    t[e >> 6][e & 63] = u;
  }
  __syncthreads();
  // the tile in its own order is X (wide) or X^T (tall); the other one gets the transposed tile
  _Float16* X = (_Float16*)(ws + L.x());
  _Float16* XT = (_Float16*)(ws + L.xt(0));
  _Float16* Xlo = (_Float16*)(ws + L.xlo());
  _Float16* same = tall ? XT : X;
  _Float16* other = tall ? X : XT;
  const int64_t ks = tall ? L.rp : L.cp, ko = tall ? L.cp : L.rp;
  for (int e = threadIdx.x; e < 64 * 16; e += 256) {
    const int a = e >> 4, b = (e & 15) * 4;
    half4 hi, lo;
    float v[4] = {t[a][b], t[a][b + 1], t[a][b + 2], t[a][b + 3]};
    split_n<4>(v, (_Float16*)&hi, (_Float16*)&lo);
    _Float16* d = same + at<W>(i0 + a, ks, j0 + b);
    *(half4*)d = hi;
    if (W == 2) *(half4*)(d + 32) = lo;
    else if (!tall) *(half4*)(Xlo + (i0 + a) * ks + j0 + b) = lo;
    float u[4] = {t[b][a], t[b + 1][a], t[b + 2][a], t[b + 3][a]};
    split_n<4>(u, (_Float16*)&hi, (_Float16*)&lo);
    d = other + at<W>(j0 + a, ko, i0 + b);
    *(half4*)d = hi;
    if (W == 2) *(half4*)(d + 32) = lo;
    else if (tall) *(half4*)(Xlo + (j0 + a) * ko + i0 + b) = lo;
  }
}

// ---- the products -------------------------------------------------------------------------------------------------
enum { PHASE_A = 0, PHASE_B = 1, PHASE_X = 2, PHASE_LAST = 3 };

// 16 bytes per lane, global -> LDS: scalar base and 32-bit offset per lane
__device__ __forceinline__ void lds_dma16_s(const char* base, uint32_t off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_addr)
               : "memory", "m0");
}

// One TILE x TILE tile of P Q^T per block.  WM x WN: a wave's part.  A stage is 128 bytes of every row (64 values, or
// 32 hi and 32 lo), brought to LDS by DMA; the 16-byte chunk c of row i lies at c ^ (i & 7), which makes the fragment
// reads (8 lanes = 8 rows, one chunk) free of bank conflicts.  NBUF stages form a ring, NBUF - 1 of them in flight.
template <int TILE, int WM, int WN, int NBUF, int W, int PHASE>
__global__ __launch_bounds__((TILE / WM) * (TILE / WN) * 64) void ns_product_kernel(
    NsArgs A, NsStep S, float ca, float cb, float cc, int parity, int bf16) {
  constexpr int NWM = TILE / WM, NWN = TILE / WN, NW = NWM * NWN, NT = NW * 64;
  constexpr int STAGE = 2 * TILE * 128;          // bytes
  constexpr int LOADS = STAGE / (NW * 1024);     // DMA instructions per wave and stage
  constexpr int FM = WM / 16, FN = WN / 16;
  constexpr int SLAB = 64 * (TILE + 1) * 4;
  __shared__ __attribute__((aligned(1024))) char lds[NBUF * STAGE > SLAB ? NBUF * STAGE : SLAB];

  // blocks b, b + 8, ... share an XCD: give each XCD a run of neighbouring tiles
  int blk = blockIdx.x;
  {
    const int nblk = gridDim.x, per = nblk / 8, rest = nblk % 8, x = blk & 7;
    blk = x * per + (x < rest ? x : rest) + (blk >> 3);
  }
  const int ii = find_item(A, blk);
  const NsItem it = A.it[ii];
  const NsLayout L(it.rows, it.cols, TILE, W);
  const int nr = L.rp / TILE, nc = L.cp / TILE;
  int q = blk - A.blk0[ii], ti, tj;
  const int per = PHASE <= PHASE_B ? nr * (nr + 1) / 2 : nr * nc;
  const int k = q / per;
  q -= k * per;
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
  char* ws = it.ws + k * L.bytes();
  const _Float16* P = (const _Float16*)(ws + (PHASE == PHASE_A ? L.x() : PHASE == PHASE_B ? L.a() : L.b()));
  const _Float16* Q = PHASE <= PHASE_B ? P : (const _Float16*)(ws + L.xt(parity));
  const int K = PHASE == PHASE_A ? L.cp : L.rp;
  const int64_t ldb = (int64_t)K * W * 2;        // bytes between rows
  const int stages = K * W / 64;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
  // loads: instruction l of a wave brings rows 8 (l NW + wave) .. + 7 of [P tile; Q tile]
  const char* pb = (const char*)P + (int64_t)ti * TILE * ldb;
  const char* qb = (const char*)Q + (int64_t)tj * TILE * ldb;
  uint32_t off[LOADS];
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    const int row = (8 * (l * NW + wave) + (lane >> 3)) % TILE;
    off[l] = (uint32_t)(row * ldb) + (((lane & 7) ^ (lane >> 3)) << 4);
  }
  const auto issue = [&](int s) {
    const uint32_t dst = lds0 + (s % NBUF) * STAGE + wave * 1024;
#pragma unroll
    for (int l = 0; l < LOADS; ++l)
      lds_dma16_s((l * NW * 8 < TILE ? pb : qb) + (int64_t)s * 128, off[l], dst + l * NW * 1024);
  };
  static_assert((TILE / 8) % NW == 0, "an instruction loads rows of one operand for every wave");

  floatx4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int frow = lane & 15, fchunk = ((lane >> 4) ^ (lane & 7)) << 4;
  for (int s = 0; s < NBUF - 1 && s < stages; ++s) issue(s);
  for (int s = 0; s < stages; ++s) {
    // stage s has arrived once only the loads issued after it are outstanding; all waves are then past stage s - 1
    if (s + NBUF - 2 < stages) wait_vm_barrier<(NBUF - 2) * LOADS>();
    else wait_vm_barrier<0>();
    if (s + NBUF - 1 < stages) issue(s + NBUF - 1);
    const char* pa = lds + (s % NBUF) * STAGE + (wm * WM + frow) * 128;
    const char* pq = lds + (s % NBUF) * STAGE + (TILE + wn * WN + frow) * 128;
    half8 a0[FM], a1[FM], b0[FN], b1[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) a0[i] = *(const half8*)(pa + i * 2048 + fchunk);
#pragma unroll
    for (int j = 0; j < FN; ++j) b0[j] = *(const half8*)(pq + j * 2048 + fchunk);
#pragma unroll
    for (int j = 0; j < FN; ++j) b1[j] = *(const half8*)(pq + j * 2048 + (fchunk ^ 64));
#pragma unroll
    for (int i = 0; i < FM; ++i) a1[i] = *(const half8*)(pa + i * 2048 + (fchunk ^ 64));
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0[i], b0[j], acc[i][j], 0, 0, 0);
    if (W == 2) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0[i], b1[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1[i], W == 2 ? b0[j] : b1[j], acc[i][j], 0, 0, 0);
  }
  __syncthreads();

  // epilogue: 64 rows at a time through LDS in fp32 (odd row length: columns are read without conflicts too)
  constexpr int LD = TILE + 1;
  float* slab = (float*)lds;
  _Float16* X = (_Float16*)(ws + L.x());
  _Float16* XT = (_Float16*)(ws + L.xt(parity ^ 1));
  _Float16* Xlo = (_Float16*)(ws + L.xlo());
  _Float16* D = (_Float16*)(ws + (PHASE == PHASE_A ? L.a() : L.b()));
  const bool tall = it.rows > it.cols;
  char* out = PHASE == PHASE_LAST ? (char*)it.p + k * it.bsp * (bf16 ? 2 : 4) : nullptr;
  const float decay = PHASE == PHASE_LAST && it.m ? (S.hyper ? S.hyper[0] : S.decay) : 0.f;
  const float gain = PHASE == PHASE_LAST ? (it.m ? (S.hyper ? S.hyper[1] : S.neg_lr) * it.scale : 1.f) * kDescale : 0.f;
  const auto put = [&](int row, int col, float v) {   // row, col of the caller's matrix
    const int64_t e = (int64_t)row * it.ldp + col;
    v *= gain;
    if (it.m) v = __builtin_fmaf(load1(out, e, bf16), decay, v);
    store1(out, e, bf16, v);
  };
  for (int s = 0; s < TILE / 64; ++s) {
    if (s) __syncthreads();
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = wm * WM + i * 16 - s * 64;
      if (row >= 0 && row < 64) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            slab[(row + (lane >> 4) * 4 + e) * LD + wn * WN + j * 16 + frow] = acc[i][j][e] * kDescale;
      }
    }
    __syncthreads();
    const int i0 = ti * TILE + s * 64, j0 = tj * TILE;
    for (int e = threadIdx.x; e < 64 * TILE / 4; e += NT) {
      const int i = e / (TILE / 4), j = e % (TILE / 4) * 4;
      float v[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) v[z] = slab[i * LD + j + z];
      half4 hi, lo;
      if (PHASE == PHASE_B) {
        const _Float16* d = P + at<W>(i0 + i, K, j0 + j);
        hi = *(const half4*)d;
        if (W == 2) lo = *(const half4*)(d + 32);
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = __builtin_fmaf(cb, W == 2 ? (float)hi[z] + (float)lo[z] : (float)hi[z], cc * v[z]);
      } else if (PHASE >= PHASE_X) {
        _Float16* d = X + at<W>(i0 + i, L.cp, j0 + j);
        hi = *(const half4*)d;
        lo = *(const half4*)(W == 2 ? d + 32 : Xlo + (int64_t)(i0 + i) * L.cp + j0 + j);
#pragma unroll
        for (int z = 0; z < 4; ++z) v[z] = __builtin_fmaf(ca, (float)hi[z] + (float)lo[z], v[z]);
      }
      if (PHASE != PHASE_A) {
#pragma unroll
        for (int z = 0; z < 4; ++z) slab[i * LD + j + z] = v[z];
      }
      if (PHASE == PHASE_LAST) {
        if (!tall && i0 + i < it.rows) {
#pragma unroll
          for (int z = 0; z < 4; ++z)
            if (j0 + j + z < it.cols) put(i0 + i, j0 + j + z, v[z]);
        }
      } else {
        split_n<4>(v, (_Float16*)&hi, (_Float16*)&lo);
        _Float16* d = PHASE == PHASE_X ? X + at<W>(i0 + i, L.cp, j0 + j) : D + at<W>(i0 + i, L.rp, j0 + j);
        *(half4*)d = hi;
        if (W == 2) *(half4*)(d + 32) = lo;
        else if (PHASE == PHASE_X) *(half4*)(Xlo + (int64_t)(i0 + i) * L.cp + j0 + j) = lo;
      }
    }
    // the other order: X^T, the mirrored triangle, or a tall result
    if (PHASE <= PHASE_B && ti == tj) continue;
    if (PHASE == PHASE_LAST && !tall) continue;
    __syncthreads();
    for (int e = threadIdx.x; e < 64 * TILE / 8; e += NT) {
      const int j = e >> 3, i = (e & 7) * 8;
      float v[8];
#pragma unroll
      for (int z = 0; z < 8; ++z) v[z] = slab[(i + z) * LD + j];
      if (PHASE == PHASE_LAST) {
        if (j0 + j < it.rows) {
#pragma unroll
          for (int z = 0; z < 8; ++z)
            if (i0 + i + z < it.cols) put(j0 + j, i0 + i + z, v[z]);
        }
      } else {
        half8 hi, lo;
        split_n<8>(v, (_Float16*)&hi, (_Float16*)&lo);
        _Float16* d = (PHASE == PHASE_X ? XT : D) + at<W>(j0 + j, L.rp, i0 + i);
        *(half8*)d = hi;
        if (W == 2) *(half8*)(d + 32) = lo;
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
struct NsPlan {
  int tile, w;
};

// Tile and operand width of each matrix.  A large tile reads its operands fewer times but there are fewer of them: a
// size is taken by the matrices that do not leave half a tile empty, if together they have a block for 3 of 4 CUs.
void ns_plan(int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec, NsPlan* plan) {
  for (int i = 0; i < n; ++i) plan[i].tile = 0;
  for (int t = 256; t >= 64; t /= 2) {
    int64_t blocks = 0;
    const auto fits = [&](int i) {
      const int64_t r = rows[i] < cols[i] ? rows[i] : cols[i];
      return plan[i].tile == 0 && (t == 64 || r > t / 2);
    };
    for (int i = 0; i < n; ++i)
      if (fits(i)) blocks += batch[i] * ((rows[i] + t - 1) / t) * ((cols[i] + t - 1) / t);
    for (int i = 0; i < n; ++i)
      if (fits(i) && (t == 64 || blocks >= 192)) plan[i] = NsPlan{t, t == 64 || prec == 0 ? 2 : 1};
  }
}

int ns_check(const char* fn, int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, int prec) {
  MMS_REQUIRE(n >= 0 && n <= 4096, fn, "0 to 4096 matrices");
  MMS_REQUIRE(n == 0 || (batch && rows && cols), fn, "null size table");
  MMS_REQUIRE(prec == 0 || prec == 1, fn, "prec 0 (split fp16) or 1 (fp16)");
  for (int i = 0; i < n; ++i)
    MMS_REQUIRE(batch[i] >= 0 && rows[i] >= 0 && cols[i] >= 0 && batch[i] <= (1 << 20) && rows[i] <= (1 << 20) &&
                    cols[i] <= (1 << 20) && batch[i] * ((rows[i] + 63) / 64) * ((cols[i] + 63) / 64) <= (1 << 28),
                fn, "matrix sizes up to 2^20 a side and 2^28 64 x 64 tiles");
  return 0;
}

template <int TILE, int WM, int WN, int NBUF, int W>
void launch_products(const NsArgs& gram, const NsArgs& full, const NsStep& S, int steps, float a, float b, float c,
                     int bf16, hipStream_t s) {
  constexpr int NT = (TILE / WM) * (TILE / WN) * 64;
  for (int i = 0; i < steps; ++i) {
    hipLaunchKernelGGL((ns_product_kernel<TILE, WM, WN, NBUF, W, PHASE_A>), dim3(gram.blk0[gram.n]), dim3(NT), 0, s,
                       gram, S, a, b, c, i & 1, bf16);
    hipLaunchKernelGGL((ns_product_kernel<TILE, WM, WN, NBUF, W, PHASE_B>), dim3(gram.blk0[gram.n]), dim3(NT), 0, s,
                       gram, S, a, b, c, i & 1, bf16);
    if (i + 1 < steps)
      hipLaunchKernelGGL((ns_product_kernel<TILE, WM, WN, NBUF, W, PHASE_X>), dim3(full.blk0[full.n]), dim3(NT), 0, s,
                         full, S, a, b, c, i & 1, bf16);
    else
      hipLaunchKernelGGL((ns_product_kernel<TILE, WM, WN, NBUF, W, PHASE_LAST>), dim3(full.blk0[full.n]), dim3(NT), 0,
                         s, full, S, a, b, c, i & 1, bf16);
  }
}

int ns_run(const char* fn, int n, const int64_t* batch, const int64_t* rows, const int64_t* cols, void* const* p,
           const int64_t* ldp, const int64_t* bsp, const void* const* g, const int64_t* ldg, const int64_t* bsg,
           float* const* m, const float* scale, int bf16, int prec, int steps, float a, float b, float c,
           const NsStep& S, void* ws, int64_t ws_bytes, void* stream) {
  MMS_REQUIRE(steps >= 1 && steps <= 64, fn, "1 to 64 steps");
  MMS_REQUIRE(S.eps > 0.0, fn, "eps must be positive");
  MMS_REQUIRE(n == 0 || (p && ldp && bsp && g && ldg && bsg), fn, "null pointer table");
  int64_t need = 0;
  const int rc = mms_muon_workspace(n, batch, rows, cols, prec, &need);
  if (rc) return rc;
  for (int i = 0; i < n; ++i) {
    if (batch[i] * rows[i] * cols[i] == 0) continue;
    MMS_REQUIRE(p[i] && g[i], fn, "null matrix");
    MMS_REQUIRE(ldp[i] >= cols[i] && ldg[i] >= cols[i] && ldp[i] < (1LL << 31) && ldg[i] < (1LL << 31), fn,
                "leading dimensions must hold a row");
    MMS_REQUIRE(bsp[i] >= 0 && bsg[i] >= 0 && (batch[i] == 1 || bsp[i] >= rows[i] * ldp[i] - (ldp[i] - cols[i])), fn,
                "stacked matrices must not overlap");
  }
  MMS_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 255) == 0), fn,
              "workspace too small (mms_muon_workspace) or not 256-byte aligned");
  hipStream_t s = mms::as_stream(stream);
  char* next = (char*)ws;
  static thread_local NsPlan plan[4096];
  ns_plan(n, batch, rows, cols, prec, plan);
  for (int tile = 256; tile >= 64; tile /= 2) {
    for (int first = 0; first < n;) {
      // the next matrices of this tile that one launch holds
      NsArgs sq{}, pack{}, gram{}, full{};
      int64_t end[4] = {0, 0, 0, 0};
      int w = 0, i = first;
      for (; i < n && sq.n < kNsItems; ++i) {
        if (plan[i].tile != tile || batch[i] * rows[i] * cols[i] == 0) continue;
        w = plan[i].w;
        const NsLayout L((int)rows[i], (int)cols[i], tile, w);
        const int64_t nb = mms::grid_for(rows[i] * cols[i], kNormElems, kNormBlocks), nr = L.rp / tile, nc = L.cp / tile;
        const int64_t add[4] = {batch[i] * nb, batch[i] * (L.rp / 64) * (L.cp / 64), batch[i] * (nr * (nr + 1) / 2),
                                batch[i] * nr * nc};
        if (sq.n && (end[1] + add[1] > (1LL << 30) || end[0] + add[0] > (1LL << 30))) break;
        const NsItem it{g[i], m ? m[i] : nullptr, p[i], next, bsg[i], bsp[i], (int)ldg[i], (int)ldp[i], (int)rows[i],
                        (int)cols[i], (int)batch[i], scale ? scale[i] : 1.f};
        next += batch[i] * L.bytes();
        int z = 0;
        for (NsArgs* A : {&sq, &pack, &gram, &full}) {
          A->it[A->n] = it;
          A->blk0[A->n] = (int)end[z];
          end[z] += add[z];
          A->blk0[++A->n] = (int)end[z++];
        }
      }
      first = i;
      if (sq.n == 0) continue;
      hipLaunchKernelGGL(muon_momentum_kernel, dim3(sq.blk0[sq.n]), dim3(256), 0, s, sq, S, bf16, tile, w);
      if (w == 2) hipLaunchKernelGGL((ns_pack_kernel<2>), dim3(pack.blk0[pack.n]), dim3(256), 0, s, pack, S, bf16, tile);
      else hipLaunchKernelGGL((ns_pack_kernel<1>), dim3(pack.blk0[pack.n]), dim3(256), 0, s, pack, S, bf16, tile);
      if (tile == 256 && w == 2) launch_products<256, 128, 64, 2, 2>(gram, full, S, steps, a, b, c, bf16, s);
      else if (tile == 256) launch_products<256, 128, 64, 2, 1>(gram, full, S, steps, a, b, c, bf16, s);
      else if (tile == 128 && w == 2) launch_products<128, 64, 64, 2, 2>(gram, full, S, steps, a, b, c, bf16, s);
      else if (tile == 128) launch_products<128, 64, 64, 2, 1>(gram, full, S, steps, a, b, c, bf16, s);
      else launch_products<64, 32, 32, 8, 2>(gram, full, S, steps, a, b, c, bf16, s);
      const int e = mms::check_launch(fn);
      if (e) return e;
    }
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
  static thread_local NsPlan plan[4096];
  ns_plan(n, batch, rows, cols, prec, plan);
  *bytes = 0;
  for (int i = 0; i < n; ++i)
    if (batch[i] * rows[i] * cols[i] > 0)
      *bytes += batch[i] * NsLayout((int)rows[i], (int)cols[i], plan[i].tile, plan[i].w).bytes();
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
  const NsStep S{(float)momentum, (float)(1.0 - momentum), nesterov, sumsq, max_norm, hyper, decay, neg_lr, eps};
  return ns_run(fn, n, batch, rows, cols, p, ldp, bsp, g, ldg, bsg, m, scale, bf16, prec, steps, a, b, c, S, ws,
                ws_bytes, stream);
}
