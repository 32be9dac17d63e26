// Learned row tables: out[i, :] = scale table[ids[i], :], and the table's gradient
//   dtable[v, :] = scale sum_{i : ids[i] = v} dout[i, :]      (indices outside the table and padding_idx: none).
//
// Both are bound by memory: the forward reads each row that occurs and writes n rows; the gradient reads n rows and
// writes all of the table's.  The gradient sorts the indices (stable, so the sums' order and with it every bit of the
// result is the same on each call), cuts the sorted list into runs of equal length whatever the indices are -- one
// that occurs in half of the positions is spread over as many runs -- and sums each run in fp32 in one walk.  Rows
// that lie inside a run are finished there; the pieces of a row that crosses runs go to the workspace and a second
// launch adds them in order.  Rows that do not occur are found by a search in the sorted list and written as zeros by
// further blocks of the same launch, so nothing is written twice.
#include "common.h"

namespace {

typedef __bf16 bf16_t;

template <typename T> struct Vec16 { static constexpr int N = 16 / sizeof(T); };

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

struct Ids {
  const void* p;
  int64_t stride;
  int is64;
  int64_t rows;      // valid indices: 0 .. rows - 1
  int64_t pad;       // index without gradient, or -1
};

__device__ __forceinline__ int64_t id_at(const Ids& I, int64_t i) {
  return I.is64 ? ((const int64_t*)I.p)[i * I.stride] : (int64_t)((const int32_t*)I.p)[i * I.stride];
}
// sort key: the row, or `rows` (behind all of them) where there is no gradient
__device__ __forceinline__ uint32_t key_at(const Ids& I, int64_t i) {
  const int64_t v = id_at(I, i);
  return v < 0 || v >= I.rows || v == I.pad ? (uint32_t)I.rows : (uint32_t)v;
}

// ---- lookup -------------------------------------------------------------------------------------------------------
// `lanes` threads (a power of two, at most 256) per row segment of lanes * N elements; blockIdx.y: the segment.
template <typename T, int N>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(Ids I, int64_t n, const T* __restrict__ table, int64_t ldt,
                                                            int dim, int lanes_log2, float scale, T* __restrict__ out,
                                                            int64_t ldo) {
  const int lane = threadIdx.x & ((1 << lanes_log2) - 1), team = threadIdx.x >> lanes_log2;
  const int64_t i = (int64_t)blockIdx.x * (256 >> lanes_log2) + team;
  const int c = ((int)blockIdx.y << lanes_log2 | lane) * N;
  if (i >= n || c >= dim) return;
  const int64_t v = id_at(I, i);
  Pack<T, N> x{};
  if (v >= 0 && v < I.rows) {
    x = *(const Pack<T, N>*)(table + v * ldt + c);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      float y = (float)x.v[q] * scale;
      asm("" : "+v"(y));   // rounded to fp32 before fp16 (not v_fma_mixlo's one rounding): the bits of the same product in torch
      x.v[q] = (T)y;
    }
  }
  *(Pack<T, N>*)(out + i * ldo + c) = x;
}

// ---- stable sort of (row, position) pairs ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = 16;
constexpr int kMaxBits = 10;                       // of a digit
constexpr int kTileRounds = 4;                     // a block of the many-block sort takes 4096 pairs
constexpr int kOneRounds = 12;                     // up to 12288 pairs are sorted by one block
constexpr int kScanBlocks = 64;                    // more blocks than this: their counts are scanned by a launch

struct SortShared {
  uint16_t cnt[kSortWaves][1 << kMaxBits];         // pairs of each digit that a wave has seen, then of the waves before
  uint32_t base[1 << kMaxBits];
  uint32_t wsum[kSortWaves];
};

// exclusive scan over the block's threads (thread t holds v of digit t)
__device__ __forceinline__ uint32_t block_scan(uint32_t v, SortShared& S) {
  uint32_t x = v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) S.wsum[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += S.wsum[w];
  __syncthreads();
  return before + x - v;
}

// The rank of each of a thread's pairs among the block's pairs of the same digit.  Wave w holds the pairs
// [w R 64, (w + 1) R 64) of the block, round j the 64 from j 64 on, so (wave, round, lane) is their order.
template <int R>
__device__ __forceinline__ void rank_pairs(const uint32_t (&digit)[R], const bool (&live)[R], int rounds, int bits,
                                           uint32_t (&rank)[R], SortShared& S) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = lane; d < (1 << bits); d += 64) S.cnt[wave][d] = 0;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (j < rounds) {
      uint64_t same = __ballot(live[j]);
      for (int b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((digit[j] >> b) & 1);
        same &= (digit[j] >> b) & 1 ? m : ~m;
      }
      const uint64_t before = same & ((1ull << lane) - 1);
      volatile uint16_t* c = &S.cnt[wave][live[j] ? digit[j] : 0];
      const uint32_t seen = *c;
      rank[j] = seen + __popcll(before);
      __builtin_amdgcn_wave_barrier();
      if (live[j] && before == 0) *c = (uint16_t)(seen + __popcll(same));
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
}

// counts of each wave -> pairs of that digit in the waves before it; returns the block's total of digit threadIdx.x
__device__ __forceinline__ uint32_t waves_before(int bits, SortShared& S) {
  uint32_t total = 0;
  if (threadIdx.x < (1u << bits))
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = S.cnt[w][threadIdx.x];
      S.cnt[w][threadIdx.x] = (uint16_t)total;
      total += c;
    }
  return total;
}

// n <= kOneRounds * 1024 pairs by one block, all digits
__global__ __launch_bounds__(kSortThreads) void sort_one_kernel(Ids I, int n, int bits, int passes,
                                                                uint2* __restrict__ out) {
  __shared__ SortShared S;
  __shared__ uint2 buf[kOneRounds * kSortThreads];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rounds = (n + kSortThreads - 1) / kSortThreads;
  uint2 p[kOneRounds];
  uint32_t digit[kOneRounds], rank[kOneRounds];
  bool live[kOneRounds];
#pragma unroll
  for (int j = 0; j < kOneRounds; ++j) {
    const int i = (wave * rounds + j) * 64 + lane;
    live[j] = j < rounds && i < n;
    p[j] = live[j] ? uint2{key_at(I, i), (uint32_t)i} : uint2{0, 0};
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
#pragma unroll
    for (int j = 0; j < kOneRounds; ++j) digit[j] = (p[j].x >> shift) & ((1u << bits) - 1);
    rank_pairs<kOneRounds>(digit, live, rounds, bits, rank, S);
    const uint32_t total = waves_before(bits, S);
    const uint32_t base = block_scan(total, S);
    if (threadIdx.x < (1u << bits)) S.base[threadIdx.x] = base;
    __syncthreads();
    const bool last = pass + 1 == passes;
#pragma unroll
    for (int j = 0; j < kOneRounds; ++j)
      if (live[j]) (last ? out : buf)[S.base[digit[j]] + S.cnt[wave][digit[j]] + rank[j]] = p[j];
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOneRounds; ++j)
      if (live[j]) p[j] = buf[(wave * rounds + j) * 64 + lane];
    __syncthreads();
  }
}

// counts[block][digit] of the block's 4096 pairs; in == null: the pairs are (key of ids[i], i)
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Ids I, const uint2* __restrict__ in, int64_t n,
                                                                  int bits, int shift, uint32_t* __restrict__ counts) {
  __shared__ uint32_t hist[1 << kMaxBits];
  if (threadIdx.x < (1u << bits)) hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kTileRounds * kSortThreads;
#pragma unroll
  for (int j = 0; j < kTileRounds; ++j) {
    const int64_t i = i0 + j * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[((in ? in[i].x : key_at(I, i)) >> shift) & ((1u << bits) - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < (1u << bits)) counts[((int64_t)blockIdx.x << bits) + threadIdx.x] = hist[threadIdx.x];
}

// counts[block][digit] -> pairs of that digit in the blocks before, totals[digit]: a block per digit
__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(uint32_t* __restrict__ counts, int nblk, int bits,
                                                                 uint32_t* __restrict__ totals) {
  __shared__ SortShared S;
  uint32_t before = 0;
  for (int b0 = 0; b0 < nblk; b0 += kSortThreads) {
    const int b = b0 + threadIdx.x;
    uint32_t* c = counts + ((int64_t)b << bits) + blockIdx.x;
    const uint32_t v = b < nblk ? *c : 0;
    const uint32_t x = block_scan(v, S) + before;
    if (b < nblk) *c = x;
    if (threadIdx.x == kSortThreads - 1) S.base[0] = x + v;
    __syncthreads();
    before = S.base[0];
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(Ids I, const uint2* __restrict__ in, int64_t n,
                                                                    int bits, int shift,
                                                                    const uint32_t* __restrict__ counts,
                                                                    const uint32_t* __restrict__ totals,
                                                                    uint2* __restrict__ out) {
  __shared__ SortShared S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)blockIdx.x * kTileRounds * kSortThreads + wave * kTileRounds * 64 + lane;
  uint2 p[kTileRounds];
  uint32_t digit[kTileRounds], rank[kTileRounds];
  bool live[kTileRounds];
#pragma unroll
  for (int j = 0; j < kTileRounds; ++j) {
    const int64_t i = i0 + j * 64;
    live[j] = i < n;
    p[j] = !live[j] ? uint2{0, 0} : in ? in[i] : uint2{key_at(I, i), (uint32_t)i};
    digit[j] = (p[j].x >> shift) & ((1u << bits) - 1);
  }
  rank_pairs<kTileRounds>(digit, live, kTileRounds, bits, rank, S);
  waves_before(bits, S);
  uint32_t total = 0, before = 0;
  if (threadIdx.x < (1u << bits)) {
    if (totals) {
      total = totals[threadIdx.x];
      before = counts[((int64_t)blockIdx.x << bits) + threadIdx.x];
    } else {
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const uint32_t c = counts[((int64_t)b << bits) + threadIdx.x];
        if (b < (int)blockIdx.x) before += c;
        total += c;
      }
    }
  }
  const uint32_t base = block_scan(total, S);
  if (threadIdx.x < (1u << bits)) S.base[threadIdx.x] = base + before;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kTileRounds; ++j)
    if (live[j]) out[S.base[digit[j]] + S.cnt[wave][digit[j]] + rank[j]] = p[j];
}

// ---- sums ---------------------------------------------------------------------------------------------------------
struct Grad {
  const uint2* sorted;    // (row, position), rows ascending; row == rows: no gradient
  int64_t n;
  int64_t rows;
  int dim, lanes_log2, run;
  int64_t nruns;
  float scale;
  int accumulate;
  float* part;            // [nruns][2][dim]: a run's piece of a row that began before it, and of one that goes on
};

// first position in the sorted list whose row is >= v
__device__ __forceinline__ int64_t lower_row(const Grad& G, uint32_t v) {
  int64_t lo = 0, hi = G.n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (G.sorted[mid].x < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename T, int N>
__device__ __forceinline__ void put_row(const Grad& G, T* g, const float (&acc)[N]) {
  Pack<T, N> x;
  if (G.accumulate) {
    x = *(const Pack<T, N>*)g;
#pragma unroll
    for (int q = 0; q < N; ++q) x.v[q] = (T)__builtin_fmaf(G.scale, acc[q], (float)x.v[q]);
  } else {
#pragma unroll
    for (int q = 0; q < N; ++q) x.v[q] = (T)(G.scale * acc[q]);
  }
  *(Pack<T, N>*)g = x;
}

constexpr int kZeroRows = 64;   // rows that a block looks up and clears

// blocks [0, sum_blocks): a team of lanes per run and column segment (blockIdx.y); the others clear absent rows
template <typename T, int N>
__global__ __launch_bounds__(256) void embedding_sum_kernel(Grad G, int64_t sum_blocks, const T* __restrict__ dout,
                                                            int64_t ldd, T* __restrict__ dtable, int64_t ldg) {
  if (blockIdx.x >= sum_blocks) {
    __shared__ bool present[kZeroRows];
    const int64_t r0 = (blockIdx.x - sum_blocks) * kZeroRows;
    const int nr = G.rows - r0 < kZeroRows ? (int)(G.rows - r0) : kZeroRows;
    if ((int)threadIdx.x < nr) {
      const uint32_t v = (uint32_t)(r0 + threadIdx.x);
      const int64_t at = lower_row(G, v);
      present[threadIdx.x] = at < G.n && G.sorted[at].x == v;
    }
    __syncthreads();
    const int c0 = (int)blockIdx.y * N << G.lanes_log2, c1 = min(G.dim, c0 + (N << G.lanes_log2));
    const int per = (c1 - c0) / N;
    const Pack<T, N> zero{};
    for (int e = threadIdx.x; e < nr * per; e += 256) {
      const int r = e / per;
      if (!present[r]) *(Pack<T, N>*)(dtable + (r0 + r) * ldg + c0 + (e - r * per) * N) = zero;
    }
    return;
  }
  const int lane = threadIdx.x & ((1 << G.lanes_log2) - 1), team = threadIdx.x >> G.lanes_log2;
  const int64_t run = (int64_t)blockIdx.x * (256 >> G.lanes_log2) + team;
  const int c = ((int)blockIdx.y << G.lanes_log2 | lane) * N;
  if (run >= G.nruns || c >= G.dim) return;
  const int64_t i0 = run * G.run, i1 = i0 + G.run < G.n ? i0 + G.run : G.n;
  float acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = 0.f;
  uint32_t cur = G.sorted[i0].x;
  bool began = i0 == 0 || G.sorted[i0 - 1].x != cur;   // the current row's first position lies in this run
  const auto flush = [&](bool ended) {
    if (cur >= G.rows) return;
    if (began && ended) {
      put_row<T, N>(G, dtable + (int64_t)cur * ldg + c, acc);
    } else {
      float* p = G.part + (run * 2 + (began ? 1 : 0)) * G.dim + c;
#pragma unroll
      for (int q = 0; q < N; ++q) p[q] = acc[q];
    }
  };
  constexpr int U = 8;
  for (int64_t i = i0; i < i1; i += U) {
    uint2 s[U];
    Pack<T, N> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = G.sorted[i + u < i1 ? i + u : i1 - 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s[u].x < G.rows) x[u] = *(const Pack<T, N>*)(dout + (int64_t)s[u].y * ldd + c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= i1) break;
      if (s[u].x != cur) {
        flush(true);
        cur = s[u].x;
        began = true;
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
      }
      if (cur >= G.rows) return;   // sorted last: nothing follows
#pragma unroll
      for (int q = 0; q < N; ++q) acc[q] += (float)x[u].v[q];
    }
  }
  flush(i1 == G.n || G.sorted[i1].x != cur);
}

// A row that crosses runs: the run where it begins adds up its pieces.  4 waves take a quarter of them each, in order.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(Grad G, T* __restrict__ dtable, int64_t ldg) {
  const int64_t run = blockIdx.x;
  const int64_t i0 = run * G.run, i1 = i0 + G.run;
  if (i1 >= G.n) return;
  const uint32_t v = G.sorted[i1 - 1].x;
  if (v >= G.rows || G.sorted[i1].x != v) return;
  if (i0 > 0 && G.sorted[i0].x == v && G.sorted[i0 - 1].x == v) return;   // began in an earlier run
  const int64_t last = (lower_row(G, v + 1) - 1) / G.run;
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (int)blockIdx.y * 64 + lane;
  // pieces: slot 1 of `run`, slot 0 of run + 1 .. last
  const int64_t count = last - run, per = (count + 3) / 4;
  float acc = 0.f;
  if (c < G.dim) {
    if (wave == 0) acc = G.part[(run * 2 + 1) * G.dim + c];
    const int64_t a = run + 1 + wave * per, b = a + per < last + 1 ? a + per : last + 1;
#pragma unroll 8
    for (int64_t k = a; k < b; ++k) acc += G.part[k * 2 * G.dim + c];
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && c < G.dim) {
    const float one[1] = {((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane]};
    put_row<T, 1>(G, dtable + (int64_t)v * ldg + c, one);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

bool aligned_rows(const void* p, int64_t ld, int dim, int dtype) {
  const int e = elem_size(dtype);
  return ((uintptr_t)p & 15) == 0 && ld * e % 16 == 0 && dim * (int64_t)e % 16 == 0;
}

// threads per row: enough 16-byte (or single-element) pieces for the row, at most a block
int lanes_for(int dim, int n) {
  int l = 0;
  while (l < 8 && ((int64_t)n << l) < dim) ++l;
  return l;
}

int check_ids(const char* fn, const void* ids, int64_t stride, int64_t n, int64_t rows, int dim, int dtype) {
  MMS_REQUIRE(dtype >= 0 && dtype <= 2, fn, "dtype 0 (fp32), 1 (bf16) or 2 (fp16)");
  MMS_REQUIRE(n >= 0 && n < (1LL << 24) && rows >= 1 && rows < (1LL << 29) && dim >= 1 && dim <= (1 << 20), fn,
              "0 to 2^24 - 1 indices, 1 to 2^29 - 1 rows of 1 to 2^20 values");
  MMS_REQUIRE(n == 0 || (ids && stride >= 0), fn, "null indices or negative stride");
  return 0;
}

struct Plan {
  int bits, passes, run, lanes_log2, vec;
  int64_t nblk, nruns, pairs, counts, part, total;   // byte offsets: pairs of the second buffer, ...
};

Plan plan_for(int64_t n, int64_t rows, int dim, int dtype, bool wide) {
  Plan p{};
  int need = 1;
  while ((rows >> need) != 0) ++need;      // keys 0 .. rows
  p.passes = (need + kMaxBits - 1) / kMaxBits;
  p.bits = (need + p.passes - 1) / p.passes;
  p.vec = wide ? 16 / elem_size(dtype) : 1;
  p.lanes_log2 = lanes_for(dim, p.vec);
  p.nblk = (n + kTileRounds * kSortThreads - 1) / (kTileRounds * kSortThreads);
  p.run = 64;
  while (p.run > 8 && (n / p.run) << p.lanes_log2 < 256 * 1024) p.run >>= 1;
  p.nruns = (n + p.run - 1) / p.run;
  const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  p.pairs = up(n * 8);
  p.counts = p.pairs * 2;
  p.part = p.counts + up((p.nblk + 1) * 4 << p.bits);
  p.total = p.part + up(p.nruns * 2 * dim * 4);
  return p;
}

template <typename T>
int launch_fwd(const Ids& I, int64_t n, const void* table, int64_t ldt, int dim, float scale, void* out, int64_t ldo,
               bool wide, hipStream_t s) {
  constexpr int V = Vec16<T>::N;
  const int vec = wide ? V : 1, l = lanes_for(dim, vec), per = 256 >> l;
  const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)((dim + (vec << l) - 1) / (vec << l)));
  if (wide)
    hipLaunchKernelGGL((embedding_fwd_kernel<T, V>), grid, dim3(256), 0, s, I, n, (const T*)table, ldt, dim, l, scale,
                       (T*)out, ldo);
  else
    hipLaunchKernelGGL((embedding_fwd_kernel<T, 1>), grid, dim3(256), 0, s, I, n, (const T*)table, ldt, dim, l, scale,
                       (T*)out, ldo);
  return 0;
}

template <typename T>
int launch_sums(const Grad& G, const Plan& p, const T* dout, int64_t ldd, T* dtable, int64_t ldg, hipStream_t s) {
  constexpr int V = Vec16<T>::N;
  const int per = 256 >> p.lanes_log2;
  const int64_t sums = (G.nruns + per - 1) / per;
  const int64_t zeros = G.accumulate ? 0 : (G.rows + kZeroRows - 1) / kZeroRows;
  const unsigned segs = (unsigned)((G.dim + (p.vec << p.lanes_log2) - 1) / (p.vec << p.lanes_log2));
  if (sums + zeros == 0) return 0;
  if (p.vec > 1)
    hipLaunchKernelGGL((embedding_sum_kernel<T, V>), dim3((unsigned)(sums + zeros), segs), dim3(256), 0, s, G, sums,
                       dout, ldd, dtable, ldg);
  else
    hipLaunchKernelGGL((embedding_sum_kernel<T, 1>), dim3((unsigned)(sums + zeros), segs), dim3(256), 0, s, G, sums,
                       dout, ldd, dtable, ldg);
  if (G.nruns > 1)
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)(G.nruns - 1), (unsigned)((G.dim + 63) / 64)),
                       dim3(256), 0, s, G, dtable, ldg);
  return 0;
}

}  // namespace

MMS_EXPORT int mms_embedding_fwd(const void* ids, int ids64, int64_t ids_stride, int64_t n, const void* table,
                                 int64_t ldt, int64_t rows, int dim, int dtype, float scale, void* out, int64_t ldo,
                                 void* stream) {
  const char* fn = "mms_embedding_fwd";
  const int rc = check_ids(fn, ids, ids_stride, n, rows, dim, dtype);
  if (rc) return rc;
  if (n == 0) return 0;
  MMS_REQUIRE(table && out && ldt >= dim && ldo >= dim, fn, "null table or output, or rows that do not fit");
  const Ids I{ids, ids_stride, ids64, rows, -1};
  const bool wide = aligned_rows(table, ldt, dim, dtype) && aligned_rows(out, ldo, dim, dtype);
  hipStream_t s = mms::as_stream(stream);
  if (dtype == 0) launch_fwd<float>(I, n, table, ldt, dim, scale, out, ldo, wide, s);
  else if (dtype == 1) launch_fwd<bf16_t>(I, n, table, ldt, dim, scale, out, ldo, wide, s);
  else launch_fwd<_Float16>(I, n, table, ldt, dim, scale, out, ldo, wide, s);
  return mms::check_launch(fn);
}

MMS_EXPORT int mms_embedding_bwd_workspace(int64_t n, int64_t rows, int dim, int dtype, int64_t* bytes) {
  const char* fn = "mms_embedding_bwd_workspace";
  const int rc = check_ids(fn, fn, 0, n, rows, dim, dtype);
  if (rc) return rc;
  MMS_REQUIRE(bytes != nullptr, fn, "null output");
  const int64_t a = plan_for(n, rows, dim, dtype, true).total, b = plan_for(n, rows, dim, dtype, false).total;
  *bytes = a > b ? a : b;
  return 0;
}

MMS_EXPORT int mms_embedding_bwd(const void* ids, int ids64, int64_t ids_stride, int64_t n, const void* dout,
                                 int64_t ldd, int64_t rows, int dim, int dtype, float scale, int64_t padding_idx,
                                 void* dtable, int64_t ldg, int accumulate, void* ws, int64_t ws_bytes, void* stream) {
  const char* fn = "mms_embedding_bwd";
  const int rc = check_ids(fn, ids, ids_stride, n, rows, dim, dtype);
  if (rc) return rc;
  MMS_REQUIRE(dtable && ldg >= dim && (n == 0 || (dout && ldd >= dim)), fn,
              "null gradients, or rows that do not fit");
  if (n == 0 && accumulate) return 0;
  const bool wide = aligned_rows(dtable, ldg, dim, dtype) && (n == 0 || aligned_rows(dout, ldd, dim, dtype));
  const Plan p = plan_for(n, rows, dim, dtype, wide);
  MMS_REQUIRE(p.total == 0 || n == 0 || (ws && ws_bytes >= p.total && ((uintptr_t)ws & 255) == 0), fn,
              "workspace too small (mms_embedding_bwd_workspace) or not 256-byte aligned");
  hipStream_t s = mms::as_stream(stream);
  const Ids I{ids, ids_stride, ids64, rows, padding_idx};
  char* w = (char*)ws;
  uint2* buf[2] = {(uint2*)w, (uint2*)(w + p.pairs)};
  uint32_t* counts = (uint32_t*)(w + p.counts);
  uint32_t* totals = counts + (p.nblk << p.bits);
  const uint2* sorted = buf[0];
  if (n > 0 && n <= kOneRounds * kSortThreads) {
    hipLaunchKernelGGL(sort_one_kernel, dim3(1), dim3(kSortThreads), 0, s, I, (int)n, p.bits, p.passes, buf[0]);
  } else if (n > 0) {
    const uint2* in = nullptr;
    for (int k = 0; k < p.passes; ++k) {
      const bool scan = p.nblk > kScanBlocks;
      hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)p.nblk), dim3(kSortThreads), 0, s, I, in, n, p.bits,
                         k * p.bits, counts);
      if (scan)
        hipLaunchKernelGGL(sort_scan_kernel, dim3(1u << p.bits), dim3(kSortThreads), 0, s, counts, (int)p.nblk, p.bits,
                           totals);
      hipLaunchKernelGGL(sort_scatter_kernel, dim3((unsigned)p.nblk), dim3(kSortThreads), 0, s, I, in, n, p.bits,
                         k * p.bits, counts, scan ? totals : nullptr, buf[k & 1]);
      in = buf[k & 1];
    }
    sorted = in;
  }
  const Grad G{sorted, n, rows, dim, p.lanes_log2, p.run, p.nruns, scale, accumulate, (float*)(w + p.part)};
  if (dtype == 0) launch_sums<float>(G, p, (const float*)dout, ldd, (float*)dtable, ldg, s);
  else if (dtype == 1) launch_sums<bf16_t>(G, p, (const bf16_t*)dout, ldd, (bf16_t*)dtable, ldg, s);
  else launch_sums<_Float16>(G, p, (const _Float16*)dout, ldd, (_Float16*)dtable, ldg, s);
  return mms::check_launch(fn);
}
