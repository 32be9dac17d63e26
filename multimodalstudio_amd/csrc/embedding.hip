// Learned row tables: out[i, :] = scale table[ids[i], :], and the table's gradient
//   dtable[v, :] = scale sum_{i : ids[i] = v} dout[i, :]      (indices outside the table and padding_idx: none).
//
// Both are bound by memory: the forward reads each row that occurs and writes n rows; the gradient reads n rows and
// writes all of the table's.  The gradient sorts the indices (stable, so the sums' order and with it every bit of the
// result is the same on each call), cuts the sorted list into runs of equal length whatever the indices are -- one
// that occurs in half of the positions is spread over as many runs -- and sums each run in fp32 in one walk.  Rows
// that lie inside a run are finished there; the pieces of a row that crosses runs go to the workspace and a second
// launch adds them in order.  Rows that do not occur are found by a search in the sorted list and written as zeros by
// further blocks of the same launch, but for the first rows, which the sort's launches clear beside their few blocks.
// Tables of at most 64 rows and calls of at most 128 positions take two launches and one.
//
// Lookup of 16384 x 4096 bf16: 32 us, 5.6 TB/s of rows written and different rows read (a copy reaches 5.1, a fill 6.8).
// Gradient of 65536 x 2048 bf16 into 131072 rows: 178 us, 4.5 TB/s of both; the sort's share of it hides behind the
// clearing of the first rows.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16_t;

// a thread's piece of a row: 16 bytes, at any element's address (the card reads and writes them unaligned)
template <typename T> struct Piece {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
// The first `count` of its values.  WHOLE: rows are whole pieces, without a branch that keeps loads from being issued
// together (65536 x 2048 bf16 into 131072 rows: 163 us against 240).
template <bool WHOLE, typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p, int count) {
  Piece<T> x;
  if (WHOLE || count >= Piece<T>::N) {
    __builtin_memcpy(&x, p, 16);
  } else {
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q) x.v[q] = q < count ? p[q] : (T)0.f;
  }
  return x;
}
// STREAM: past the caches, for an output that is larger than they are
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
template <bool WHOLE, bool STREAM = false, typename T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& x, int count) {
  if (WHOLE || count >= Piece<T>::N) {
    if (STREAM) {
      words4 w;
      __builtin_memcpy(&w, &x, 16);
      __builtin_nontemporal_store(w, (words4*)p);
    } else {
      __builtin_memcpy(p, &x, 16);
    }
  } else {
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q)
      if (q < count) p[q] = x.v[q];
  }
}

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
// A team of `lanes` threads (a power of two, at most 256) per R rows' segments of lanes pieces; blockIdx.y: the segment.
template <typename T, bool WHOLE, int R, bool STREAM>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(Ids I, int64_t n, const T* __restrict__ table, int64_t ldt,
                                                            int dim, int lanes_log2, float scale, T* __restrict__ out,
                                                            int64_t ldo) {
  constexpr int N = Piece<T>::N;
  const int lane = threadIdx.x & ((1 << lanes_log2) - 1), team = threadIdx.x >> lanes_log2;
  const int64_t i0 = ((int64_t)blockIdx.x * (256 >> lanes_log2) + team) * R;
  const int c = ((int)blockIdx.y << lanes_log2 | lane) * N;
  if (i0 >= n || c >= dim) return;
  int64_t v[R];
  Piece<T> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = id_at(I, i0 + r < n ? i0 + r : n - 1);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (v[r] >= 0 && v[r] < I.rows) x[r] = load_piece<WHOLE>(table + v[r] * ldt + c, dim - c);
    else x[r] = Piece<T>{};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (i0 + r >= n) break;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      float y = (float)x[r].v[q] * scale;
      asm("" : "+v"(y));   // rounded to fp32 before fp16 (not v_fma_mixlo's one rounding): the bits of the same product in torch
      x[r].v[q] = (T)y;
    }
    store_piece<WHOLE, STREAM>(out + (i0 + r) * ldo + c, x[r], dim - c);
  }
}

// ---- zeros in the shadow of the sort --------------------------------------------------------------------------------
// The sort keeps a few dozen blocks busy; further blocks of its launches clear the table's first rows meanwhile (rows
// that occur among those are written twice).
struct Zeros {
  char* p;              // the first byte to clear
  int64_t rows;         // rows of `bytes` bytes, `ld` apart
  int64_t bytes, ld;
  int first;            // the launch's first block that clears
  int stream;           // past the caches: a table of more than kLargeTable
};
constexpr int64_t kZeroChunk = 1 << 16;   // bytes per such block
constexpr int64_t kLargeTable = 128 << 20;   // half of the last cache

__device__ __forceinline__ bool clear_rows(const Zeros& Z) {
  if ((int)blockIdx.x < Z.first) return false;
  const bool dense = Z.ld == Z.bytes;
  const int64_t bytes = dense ? Z.rows * Z.bytes : Z.bytes, per = (bytes + 15) / 16, all = dense ? per : per * Z.rows;
  const int64_t begin = ((int64_t)blockIdx.x - Z.first) * (kZeroChunk / 16);
  const int64_t end = begin + kZeroChunk / 16 < all ? begin + kZeroChunk / 16 : all;
  const uint4 zero{0, 0, 0, 0};
  for (int64_t e = begin + threadIdx.x; e < end; e += blockDim.x) {
    const int64_t r = dense ? 0 : e / per, c = (e - r * per) * 16;
    char* p = Z.p + r * Z.ld + c;
    if (c + 16 > bytes)
      for (int64_t b = c; b < bytes; b += 2, p += 2) *(uint16_t*)p = 0;
    else if (Z.stream)
      __builtin_nontemporal_store(words4{0, 0, 0, 0}, (words4*)p);
    else
      __builtin_memcpy(p, &zero, 16);
  }
  return true;
}

// ---- stable sort of (row, position) pairs ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = 16;
constexpr int kMaxBits = 10;                       // of a digit
constexpr int kTileRounds = 2;                     // a block of the many-block sort takes 2048 pairs
constexpr int kOneRounds = 4;                      // up to 4096 pairs are sorted by one block
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
                                                                uint2* __restrict__ out, Zeros Z) {
  if (clear_rows(Z)) return;
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
      if (live[j]) {
        const uint32_t to = S.base[digit[j]] + S.cnt[wave][digit[j]] + rank[j];
        if (last) out[to] = p[j];
        else buf[to] = p[j];
      }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOneRounds; ++j)
      if (live[j]) p[j] = buf[(wave * rounds + j) * 64 + lane];
    __syncthreads();
  }
}

// counts[digit][block] of the block's 2048 pairs (rows of ld: whole uint4s); in == null: the pairs are (key of ids[i], i)
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Ids I, const uint2* __restrict__ in, int64_t n,
                                                                  int bits, int shift, uint32_t* __restrict__ counts,
                                                                  int ld, Zeros Z) {
  if (clear_rows(Z)) return;
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
  if (threadIdx.x < (1u << bits)) counts[(int64_t)threadIdx.x * ld + blockIdx.x] = hist[threadIdx.x];
}

// counts[digit][block] -> pairs of that digit in the blocks before, totals[digit]: a block per digit
__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(uint32_t* __restrict__ counts, int nblk, int ld,
                                                                 uint32_t* __restrict__ totals) {
  __shared__ SortShared S;
  uint32_t before = 0;
  for (int b0 = 0; b0 < nblk; b0 += kSortThreads) {
    const int b = b0 + threadIdx.x;
    uint32_t* c = counts + (int64_t)blockIdx.x * ld + b;
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
                                                                    const uint32_t* __restrict__ counts, int ld,
                                                                    const uint32_t* __restrict__ totals,
                                                                    uint2* __restrict__ out, int nblk, Zeros Z) {
  if (clear_rows(Z)) return;
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
  // the digit's counts of all blocks (at most kScanBlocks of them), or the scanned one
  uint32_t total = 0, before = 0;
  uint4 c[kScanBlocks / 4];
  if (!totals && threadIdx.x < (1u << bits)) {
#pragma unroll
    for (int q = 0; q < kScanBlocks / 4; ++q)
      c[q] = q * 4 < nblk ? *(const uint4*)(counts + (int64_t)threadIdx.x * ld + q * 4) : uint4{0, 0, 0, 0};
  }
  rank_pairs<kTileRounds>(digit, live, kTileRounds, bits, rank, S);
  waves_before(bits, S);
  if (threadIdx.x < (1u << bits)) {
    if (totals) {
      total = totals[threadIdx.x];
      before = counts[(int64_t)threadIdx.x * ld + blockIdx.x];
    } else {
      const int n = nblk, me = blockIdx.x;
      const auto add = [&](int b, uint32_t v) {
        total += b < n ? v : 0;
        before += b < me ? v : 0;
      };
#pragma unroll
      for (int q = 0; q < kScanBlocks / 4; ++q) {
        add(q * 4, c[q].x); add(q * 4 + 1, c[q].y); add(q * 4 + 2, c[q].z); add(q * 4 + 3, c[q].w);
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
  float* part;            // [nruns][2][part_ld]: a run's piece of a row that began before it, and of one that goes on
  int part_ld;
  int64_t cleared;        // rows below this are zeros already
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

// a finished piece of a row of the gradient, from its sum
template <typename T, bool WHOLE>
__device__ __forceinline__ void put_row(T* g, const float (&acc)[Piece<T>::N], float scale, int accumulate, int count) {
  Piece<T> x;
  if (accumulate) {
    x = load_piece<WHOLE>(g, count);
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q) x.v[q] = (T)__builtin_fmaf(scale, acc[q], (float)x.v[q]);
  } else {
#pragma unroll
    for (int q = 0; q < Piece<T>::N; ++q) x.v[q] = (T)(scale * acc[q]);
  }
  store_piece<WHOLE>(g, x, count);
}

constexpr int kZeroRows = 64;   // rows that a block looks up and clears

// blocks [0, sum_blocks): a team of lanes per run and column segment (blockIdx.y); the others clear absent rows from
// `cleared` on
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void embedding_sum_kernel(Grad G, int64_t sum_blocks, const T* __restrict__ dout,
                                                            int64_t ldd, T* __restrict__ dtable, int64_t ldg) {
  constexpr int N = Piece<T>::N;
  if (blockIdx.x >= sum_blocks) {
    __shared__ bool present[kZeroRows];
    const int64_t r0 = G.cleared + (blockIdx.x - sum_blocks) * kZeroRows;
    const int nr = G.rows - r0 < kZeroRows ? (int)(G.rows - r0) : kZeroRows;
    if ((int)threadIdx.x < nr) {
      const uint32_t v = (uint32_t)(r0 + threadIdx.x);
      const int64_t at = lower_row(G, v);
      present[threadIdx.x] = at < G.n && G.sorted[at].x == v;
    }
    __syncthreads();
    const int c0 = (int)blockIdx.y * N << G.lanes_log2, c1 = min(G.dim, c0 + (N << G.lanes_log2));
    const int per = (c1 - c0 + N - 1) / N;
    for (int e = threadIdx.x; e < nr * per; e += 256) {
      const int r = e / per, c = c0 + (e - r * per) * N;
      if (!present[r]) store_piece<WHOLE>(dtable + (r0 + r) * ldg + c, Piece<T>{}, c1 - c);
    }
    return;
  }
  const int lane = threadIdx.x & ((1 << G.lanes_log2) - 1), team = threadIdx.x >> G.lanes_log2;
  const int64_t run = (int64_t)blockIdx.x * (256 >> G.lanes_log2) + team;
  const int c = ((int)blockIdx.y << G.lanes_log2 | lane) * N;
  if (run >= G.nruns || c >= G.dim) return;
  const int left = G.dim - c;
  const int64_t i0 = run * G.run, i1 = i0 + G.run < G.n ? i0 + G.run : G.n;
  float acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = 0.f;
  uint32_t cur = G.sorted[i0].x;
  bool began = i0 == 0 || G.sorted[i0 - 1].x != cur;   // the current row's first position lies in this run
  const auto flush = [&](bool ended) {
    if (cur >= G.rows) return;
    if (began && ended) {
      put_row<T, WHOLE>(dtable + (int64_t)cur * ldg + c, acc, G.scale, G.accumulate, left);
    } else {
      float* p = G.part + (run * 2 + (began ? 1 : 0)) * G.part_ld + c;   // rows padded to whole pieces
#pragma unroll
      for (int q = 0; q < N; ++q) p[q] = acc[q];
    }
  };
  constexpr int U = 8;
  for (int64_t i = i0; i < i1; i += U) {
    uint2 s[U];
    Piece<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = G.sorted[i + u < i1 ? i + u : i1 - 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s[u].x < G.rows) x[u] = load_piece<WHOLE>(dout + (int64_t)s[u].y * ldd + c, left);
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

// A row that crosses runs: the run where it begins adds up its pieces.  4 waves take a quarter of them each, in order;
// a lane has 4 columns.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(Grad G, T* __restrict__ dtable, int64_t ldg) {
  const int64_t run = blockIdx.x;
  const int64_t i0 = run * G.run, i1 = i0 + G.run;
  if (i1 >= G.n) return;
  const uint32_t v = G.sorted[i1 - 1].x;
  if (v >= G.rows || G.sorted[i1].x != v) return;
  if (i0 > 0 && G.sorted[i0].x == v && G.sorted[i0 - 1].x == v) return;   // began in an earlier run
  __shared__ float4 red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // runs that begin with v: 64 looked at together
  int64_t count = 0;
  for (;;) {
    const int64_t at = (run + 1 + count + lane) * G.run;
    const uint64_t same = __ballot(at < G.n && G.sorted[at < G.n ? at : 0].x == v);
    count += same == ~0ull ? 64 : __builtin_ctzll(~same);
    if (same != ~0ull) break;
  }
  const int c = ((int)blockIdx.y * 64 + lane) * 4;
  // pieces: slot 1 of `run`, slot 0 of run + 1 .. run + count
  const int64_t per = (count + 3) / 4;
  float4 acc{0.f, 0.f, 0.f, 0.f};
  const auto add = [&](int64_t slot) {
    const float4 x = *(const float4*)(G.part + slot * G.part_ld + c);
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  };
  if (c < G.dim) {
    if (wave == 0) add(run * 2 + 1);
    const int64_t a = run + 1 + wave * per, b = a + per < run + 1 + count ? a + per : run + 1 + count;
#pragma unroll 8
    for (int64_t k = a; k < b; ++k) add(k * 2);
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && c < G.dim) {
    const float4 x = red[0][lane], y = red[1][lane], z = red[2][lane], w = red[3][lane];
    const float sum[4] = {((x.x + y.x) + z.x) + w.x, ((x.y + y.y) + z.y) + w.y, ((x.z + y.z) + z.z) + w.z,
                          ((x.w + y.w) + z.w) + w.w};
    T* g = dtable + (int64_t)v * ldg + c;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c + q < G.dim) g[q] = (T)(G.accumulate ? __builtin_fmaf(G.scale, sum[q], (float)g[q]) : G.scale * sum[q]);
  }
}

// ---- a table of few rows ------------------------------------------------------------------------------------------
// Blocks sort and sum 256 positions each and leave a sum per row that occurs among them; a second launch adds those
// up, block after block.  (Per-view codes, 10240 positions of 45 rows of 32 fp32 values: 12 us a call, 24 by the sort;
// the GPU is through with them in 9.)
constexpr int kFewRows = 64, kFewTile = 256, kFewBits = 7;   // keys 0 .. 64

struct Few {
  int64_t n;
  int rows, dim, lanes_log2, accumulate;
  float scale;
  int64_t blocks;
  uint32_t* present;      // [blocks][kFewRows / 32]
  float* part;            // [blocks][rows][part_ld]
  int part_ld;
};

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void few_sum_kernel(Ids I, Few F, const T* __restrict__ dout, int64_t ldd) {
  constexpr int N = Piece<T>::N;
  __shared__ uint16_t cnt[4][256];
  __shared__ uint32_t base[256];
  __shared__ uint32_t wsum[4];
  __shared__ uint16_t key[kFewTile], pos[kFewTile];
  __shared__ float cross[256 * N * 2];      // what a team's run has of a row that began before it, and of one that goes on
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = threadIdx.x;
  const int64_t i0 = (int64_t)blockIdx.x * kFewTile;
  // sort: rank among the wave's 64 positions by ballots, then the waves in order
  const uint32_t k = i0 + t < F.n ? key_at(I, i0 + t) : F.rows;    // `rows`: no gradient, sorted last
  cnt[0][t] = cnt[1][t] = cnt[2][t] = cnt[3][t] = 0;
  __syncthreads();
  uint64_t same = ~0ull;
  for (int b = 0; b < kFewBits; ++b) {
    const uint64_t m = __ballot((k >> b) & 1);
    same &= (k >> b) & 1 ? m : ~m;
  }
  const uint32_t before = __popcll(same & ((1ull << lane) - 1));
  if (before == 0) cnt[wave][k] = (uint16_t)__popcll(same);
  __syncthreads();
  const uint32_t c0 = cnt[0][t], c1 = cnt[1][t], c2 = cnt[2][t], total = c0 + c1 + c2 + cnt[3][t];
  uint32_t x = total;
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) wsum[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; ++w) x += wsum[w];
  base[t] = x - total;
  cnt[0][t] = 0; cnt[1][t] = (uint16_t)c0; cnt[2][t] = (uint16_t)(c0 + c1); cnt[3][t] = (uint16_t)(c0 + c1 + c2);
  const uint64_t there = __ballot(total != 0);
  if (t < kFewRows && (t & 31) == 0 && blockIdx.y == 0)
    F.present[blockIdx.x * (kFewRows / 32) + t / 32] =
        (uint32_t)(there >> (t & 32)) & (F.rows - t >= 32 ? ~0u : F.rows > t ? (1u << (F.rows - t)) - 1 : 0u);
  __syncthreads();
  const uint32_t at = base[k] + cnt[wave][k] + before;
  key[at] = (uint16_t)k;
  pos[at] = (uint16_t)t;
  __syncthreads();
  const int live = (int)base[F.rows];     // positions with a gradient
  // sums: a team of lanes per run of the sorted positions
  const int l = t & ((1 << F.lanes_log2) - 1), team = t >> F.lanes_log2, teams = 256 >> F.lanes_log2;
  const int c = ((int)blockIdx.y << F.lanes_log2 | l) * N, left = F.dim - c;
  const int run = kFewTile / teams, r0 = team * run, r1 = min(r0 + run, live);
  float* part = F.part + (int64_t)blockIdx.x * F.rows * F.part_ld + c;
  float acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = 0.f;
  const auto keep = [&](float* p) {
#pragma unroll
    for (int q = 0; q < N; ++q) p[q] = acc[q];
  };
  if (r0 < r1 && left > 0) {
    int cur = key[r0];
    bool began = r0 == 0 || key[r0 - 1] != cur;
    constexpr int U = 8;
    for (int i = r0; i < r1; i += U) {
      Piece<T> p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) p[u] = load_piece<WHOLE>(dout + (i0 + pos[min(i + u, r1 - 1)]) * ldd + c, left);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= r1) break;
        if (key[i + u] != cur) {
          if (began) keep(part + (int64_t)cur * F.part_ld);
          else keep(cross + t * N);
          cur = key[i + u];
          began = true;
#pragma unroll
          for (int q = 0; q < N; ++q) acc[q] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += (float)p[u].v[q];
      }
    }
    const bool ended = r1 == live || key[r1] != cur;
    if (began && ended) keep(part + (int64_t)cur * F.part_ld);
    else keep(cross + (began ? 256 * N : 0) + t * N);
  }
  __syncthreads();
  // a row that crosses runs: the team where it begins adds the others' pieces, in order
  if (r0 < r1 && left > 0 && r1 < live) {
    const int cur = key[r1 - 1];
    const bool began = r0 == 0 || key[r0] != cur || key[r0 - 1] != cur;
    if (began && key[r1] == cur) {
#pragma unroll
      for (int q = 0; q < N; ++q) acc[q] = cross[256 * N + t * N + q];
      for (int o = team + 1; o < teams && o * run < live && key[o * run] == cur; ++o)
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += cross[((o << F.lanes_log2) + l) * N + q];
      keep(part + (int64_t)cur * F.part_ld);
    }
  }
}

// blockIdx.x: a row; 64 lanes x 4 waves: a lane has a column, a wave a quarter of the blocks
template <typename T>
__global__ __launch_bounds__(256) void few_join_kernel(Few F, T* __restrict__ dtable, int64_t ldg) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x;
  const int c = (int)blockIdx.y * 64 + lane;
  const int64_t per = (F.blocks + 3) / 4, a = wave * per, b = a + per < F.blocks ? a + per : F.blocks;
  float acc = 0.f;
  bool any = false;
#pragma unroll 8
  for (int64_t k = a; k < b; ++k) {
    const bool there = F.present[k * (kFewRows / 32) + r / 32] >> (r & 31) & 1;
    // a row that does not occur in a block was not written there
    const float x = F.part[(k * F.rows + r) * F.part_ld + (c < F.dim ? c : 0)];
    acc += there ? x : 0.f;
    any |= there;
  }
  red[wave][lane] = acc;
  any = __syncthreads_or(any);
  if (wave == 0 && c < F.dim && (any || !F.accumulate)) {
    T* g = dtable + (int64_t)r * ldg + c;
    const float sum = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
    *g = (T)(F.accumulate ? __builtin_fmaf(F.scale, sum, (float)*g) : F.scale * sum);
  }
}

// ---- few positions --------------------------------------------------------------------------------------------------
// One launch and no workspace: every block reads all of the indices.  Blocks of teams sort them (each thread counts what
// lies before its own) and a team per sorted position and column segment sums a row, if it begins there; further blocks
// clear the rows of theirs that do not occur.  Launching bounds it (16 .. 128 positions: 8.5 us a call, 13 .. 16 with the
// launches of a sort and of runs).  128 positions of one row, which one team sums: 13 .. 17 us, as with those; past that
// it would be slower (256: 24).
constexpr int kBriefN = 128, kBriefRows = 4096;

struct Brief {
  int n, dim, lanes_log2, accumulate;
  float scale;
  int row_blocks, zero_rows;   // blocks of teams, and rows that each of the others clears
  int stream;
};

template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void embedding_brief_kernel(Ids I, Brief B, const T* __restrict__ dout, int64_t ldd,
                                                              T* __restrict__ dtable, int64_t ldg) {
  constexpr int N = Piece<T>::N;
  const int t = threadIdx.x;
  const uint32_t mine = t < B.n ? key_at(I, t) : (uint32_t)I.rows;
  const int c0 = (int)blockIdx.y * N << B.lanes_log2;
  if ((int)blockIdx.x >= B.row_blocks) {
    __shared__ bool present[kBriefRows];
    const int64_t r0 = (int64_t)((int)blockIdx.x - B.row_blocks) * B.zero_rows;
    const int nr = I.rows - r0 < B.zero_rows ? (int)(I.rows - r0) : B.zero_rows;
    for (int r = t; r < nr; r += 256) present[r] = false;
    __syncthreads();
    if (mine >= r0 && mine < r0 + nr) present[mine - r0] = true;
    __syncthreads();
    const int c1 = min(B.dim, c0 + (N << B.lanes_log2)), per = (c1 - c0 + N - 1) / N;
    for (int e = t; e < nr * per; e += 256) {
      const int r = e / per, c = c0 + (e - r * per) * N;
      if (present[r]) continue;
      T* p = dtable + (r0 + r) * ldg + c;
      if (B.stream) store_piece<WHOLE, true>(p, Piece<T>{}, c1 - c);
      else store_piece<WHOLE>(p, Piece<T>{}, c1 - c);
    }
    return;
  }
  __shared__ uint4 key4[kBriefN / 4];
  __shared__ uint32_t key[kBriefN];
  __shared__ int pos[kBriefN], length[kBriefN];
  if (t < kBriefN) ((uint32_t*)key4)[t] = mine;
  __syncthreads();
  int before = 0, same = 0;
  for (int q = 0; q < B.n; q += 32) {   // (what is past n has the largest key)
    uint4 k4[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) k4[u] = key4[q / 4 + u];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t k[4] = {k4[u].x, k4[u].y, k4[u].z, k4[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        before += k[e] < mine || (k[e] == mine && q + 4 * u + e < t);
        same += k[e] == mine;
      }
    }
  }
  if (t < B.n) {
    key[before] = mine;
    pos[before] = t;
    length[before] = same;
  }
  __syncthreads();
  const int team = t >> B.lanes_log2, i = (int)blockIdx.x * (256 >> B.lanes_log2) + team;
  const int c = c0 + (t & ((1 << B.lanes_log2) - 1)) * N, left = B.dim - c;
  if (i >= B.n || left <= 0) return;
  const uint32_t row = key[i];
  if (row >= I.rows || (i > 0 && key[i - 1] == row)) return;
  const int end = i + length[i];
  float acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = 0.f;
  int at = i;
  const auto some = [&](auto count) {   // rows loaded together
    constexpr int U = decltype(count)::value;
    Piece<T> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load_piece<WHOLE>(dout + (int64_t)pos[min(at + u, end - 1)] * ldd + c, left);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u < end)
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += (float)x[u].v[q];
    at += U;
  };
  while (end - at > 8) some(std::integral_constant<int, 32>{});
  while (at < end) some(std::integral_constant<int, 4>{});
  put_row<T, WHOLE>(dtable + (int64_t)row * ldg + c, acc, B.scale, B.accumulate, left);
}

// ---- host ---------------------------------------------------------------------------------------------------------
int piece_of(int dtype) { return dtype == 0 ? 4 : 8; }

// threads per row: enough pieces of `n` values for the row, at most a block
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
  bool brief, few;
  int bits, passes, run, lanes_log2, part_ld;
  int64_t nblk, nruns, pairs, counts, part, total;   // byte offsets: the pairs' second buffer, ...
};

Plan plan_for(int64_t n, int64_t rows, int dim, int dtype) {
  Plan p{};
  const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  const int N = piece_of(dtype);
  p.lanes_log2 = lanes_for(dim, N);
  p.part_ld = (dim + N - 1) / N * N;
  // Few positions: one launch.
  p.brief = n > 0 && n <= kBriefN;
  if (p.brief) return p;
  // Few rows: two launches instead of four to six, as long as the blocks' sums (rows of 256 positions) are less than the
  // positions themselves and a row's wave has no more than 64 blocks to add up.
  p.few = n > 0 && rows <= kFewRows && n <= 256 * kFewTile && dim <= 4096;
  if (p.few) {
    p.lanes_log2 = p.lanes_log2 < 5 ? p.lanes_log2 : 5;   // 8 teams or more to a block: runs of 32 positions or fewer
    p.nblk = (n + kFewTile - 1) / kFewTile;
    p.part = up(p.nblk * (kFewRows / 32) * 4);
    p.total = p.part + up(p.nblk * rows * p.part_ld * 4);
    return p;
  }
  int need = 1;
  while ((rows >> need) != 0) ++need;      // keys 0 .. rows
  p.passes = (need + kMaxBits - 1) / kMaxBits;
  p.bits = (need + p.passes - 1) / p.passes;
  p.nblk = (n + kTileRounds * kSortThreads - 1) / (kTileRounds * kSortThreads);
  // 512 blocks of teams if there are positions enough (9001 x 771: 56 us with runs of 16, 63, 78, 111 with 32, 64, 128)
  p.run = 128;
  while (p.run > 8 && (n / p.run) << p.lanes_log2 < 128 * 1024) p.run >>= 1;
  p.nruns = (n + p.run - 1) / p.run;
  p.pairs = up(n * 8);
  p.counts = p.pairs * 2;
  p.part = p.counts + up((p.nblk + 3) / 4 * 4 * 4 << p.bits) + (4 << p.bits);   // the digits' totals last
  p.total = p.part + up(p.nruns * 2 * p.part_ld * 4);
  return p;
}

template <typename T>
void launch_fwd(const Ids& I, int64_t n, const void* table, int64_t ldt, int dim, float scale, void* out, int64_t ldo,
                hipStream_t s) {
  constexpr int N = Piece<T>::N;
  // 4 rows a team once there are blocks enough (33 MB of output; 16384 x 4096 bf16: 46 us with one row a team, 42 with 4);
  // past the caches from half of the last one on.  That alone is faster always (16384 x 4096: 32 us), but what reads the
  // rows next pays for it: lookup and a product with a 4096 x 256 matrix, through the caches and past them, 64 MB of rows
  // 63.6 and 66.4 us, 128 MB 91 and 94, 256 MB 185 and 163; lookup and an elementwise pass 41.9 and 43.2, 90.5 and 84.5,
  // 177 and 174.
  const int l = lanes_for(dim, N), segs = (dim + (N << l) - 1) / (N << l);
  const bool many = (n << l) * segs >= 4 * 256 * 2048;
  const int per = (256 >> l) * (many ? 4 : 1);
  const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)segs);
  const bool stream = many && n * dim * (int64_t)sizeof(T) >= kLargeTable;
  const auto kernel =
      dim % N == 0 ? stream ? embedding_fwd_kernel<T, true, 4, true> : many ? embedding_fwd_kernel<T, true, 4, false>
                                                                            : embedding_fwd_kernel<T, true, 1, false>
                   : stream ? embedding_fwd_kernel<T, false, 4, true> : many ? embedding_fwd_kernel<T, false, 4, false>
                                                                             : embedding_fwd_kernel<T, false, 1, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, I, n, (const T*)table, ldt, dim, l, scale, (T*)out, ldo);
}

template <typename T>
void launch_few(const Ids& I, const Few& F, const void* dout, int64_t ldd, void* dtable, int64_t ldg, hipStream_t s) {
  const int seg = Piece<T>::N << F.lanes_log2;
  const auto kernel = F.dim % Piece<T>::N == 0 ? few_sum_kernel<T, true> : few_sum_kernel<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)F.blocks, (unsigned)((F.dim + seg - 1) / seg)), dim3(256), 0, s,
                     I, F, (const T*)dout, ldd);
  hipLaunchKernelGGL((few_join_kernel<T>), dim3((unsigned)F.rows, (unsigned)((F.dim + 63) / 64)), dim3(256), 0, s, F,
                     (T*)dtable, ldg);
}

template <typename T>
void launch_brief(const Ids& I, Brief B, const void* dout, int64_t ldd, void* dtable, int64_t ldg, hipStream_t s) {
  const int seg = Piece<T>::N << B.lanes_log2, teams = 256 >> B.lanes_log2;
  B.row_blocks = (B.n + teams - 1) / teams;
  const int64_t row = std::min(seg, B.dim) * (int64_t)sizeof(T);
  B.zero_rows = (int)std::min<int64_t>(kBriefRows, std::max<int64_t>(1, kZeroChunk / row));
  B.stream = I.rows * B.dim * (int64_t)sizeof(T) > kLargeTable;
  const int64_t zeros = B.accumulate ? 0 : (I.rows + B.zero_rows - 1) / B.zero_rows;
  const auto kernel = B.dim % Piece<T>::N == 0 ? embedding_brief_kernel<T, true> : embedding_brief_kernel<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(B.row_blocks + zeros), (unsigned)((B.dim + seg - 1) / seg)), dim3(256), 0, s,
                     I, B, (const T*)dout, ldd, (T*)dtable, ldg);
}

template <typename T>
void launch_sums(const Grad& G, const void* dout, int64_t ldd, void* dtable, int64_t ldg, hipStream_t s) {
  const int per = 256 >> G.lanes_log2, seg = Piece<T>::N << G.lanes_log2;
  const int64_t sums = (G.nruns + per - 1) / per;
  const int64_t zeros = G.accumulate ? 0 : (G.rows - G.cleared + kZeroRows - 1) / kZeroRows;
  const auto kernel = G.dim % Piece<T>::N == 0 ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(sums + zeros), (unsigned)((G.dim + seg - 1) / seg)),
                     dim3(256), 0, s, G, sums, (const T*)dout, ldd, (T*)dtable, ldg);
  if (G.nruns > 1)
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)(G.nruns - 1), (unsigned)((G.dim + 255) / 256)),
                       dim3(256), 0, s, G, (T*)dtable, ldg);
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
  hipStream_t s = mms::as_stream(stream);
  if (dtype == 0) launch_fwd<float>(I, n, table, ldt, dim, scale, out, ldo, s);
  else if (dtype == 1) launch_fwd<bf16_t>(I, n, table, ldt, dim, scale, out, ldo, s);
  else launch_fwd<_Float16>(I, n, table, ldt, dim, scale, out, ldo, s);
  return mms::check_launch(fn);
}

MMS_EXPORT int mms_embedding_bwd_workspace(int64_t n, int64_t rows, int dim, int dtype, int64_t* bytes) {
  const char* fn = "mms_embedding_bwd_workspace";
  const int rc = check_ids(fn, fn, 0, n, rows, dim, dtype);
  if (rc) return rc;
  MMS_REQUIRE(bytes != nullptr, fn, "null output");
  *bytes = plan_for(n, rows, dim, dtype).total;
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
  const Plan p = plan_for(n, rows, dim, dtype);
  MMS_REQUIRE(p.total == 0 || n == 0 || (ws && ws_bytes >= p.total && ((uintptr_t)ws & 255) == 0), fn,
              "workspace too small (mms_embedding_bwd_workspace) or not 256-byte aligned");
  hipStream_t s = mms::as_stream(stream);
  const Ids I{ids, ids_stride, ids64, rows, padding_idx};
  char* w = (char*)ws;
  if (p.brief) {
    const Brief B{(int)n, dim, p.lanes_log2, accumulate, scale, 0, 0, 0};
    if (dtype == 0) launch_brief<float>(I, B, dout, ldd, dtable, ldg, s);
    else if (dtype == 1) launch_brief<bf16_t>(I, B, dout, ldd, dtable, ldg, s);
    else launch_brief<_Float16>(I, B, dout, ldd, dtable, ldg, s);
    return mms::check_launch(fn);
  }
  if (p.few) {
    const Few F{n, (int)rows, dim, p.lanes_log2, accumulate, scale, p.nblk, (uint32_t*)w, (float*)(w + p.part), p.part_ld};
    if (dtype == 0) launch_few<float>(I, F, dout, ldd, dtable, ldg, s);
    else if (dtype == 1) launch_few<bf16_t>(I, F, dout, ldd, dtable, ldg, s);
    else launch_few<_Float16>(I, F, dout, ldd, dtable, ldg, s);
    return mms::check_launch(fn);
  }
  uint2* buf[2] = {(uint2*)w, (uint2*)(w + p.pairs)};
  uint32_t* counts = (uint32_t*)(w + p.counts);
  const int ld = (int)((p.nblk + 3) / 4 * 4);
  uint32_t* totals = counts + ((int64_t)ld << p.bits);
  const uint2* sorted = buf[0];
  const bool one = n <= kOneRounds * kSortThreads;
  // As much as hides in the sort's launches, in one of a single block or two for each digit (9001 indices below 50257, 771
  // wide: 70 us with nothing cleared there, 63 with 24 MB a launch, 56 with 48; 65536 below 131072, 2048 wide: 197, 192,
  // 189, and 196 with 136 MB, all of the table; past the caches 51 and 179).
  const int es = dtype == 0 ? 4 : 2, launches = one ? 1 : 2 * p.passes;
  const int64_t row_bytes = (int64_t)dim * es;
  const int64_t share = one ? ((n + kSortThreads - 1) / kSortThreads * p.passes * 5 + 10) << 20 : 48 << 20;
  int64_t cleared = accumulate || n == 0 ? 0 : launches * share / row_bytes;
  if (cleared > rows) cleared = rows;
  const int64_t each = (cleared + launches - 1) / launches;
  int64_t begun = 0;
  // the next launch's share of the rows, and its blocks behind `first` others
  const auto zeros = [&](int64_t first, unsigned& blocks) {
    Zeros Z{(char*)dtable + begun * ldg * es, begun + each < cleared ? each : cleared - begun, row_bytes, ldg * es, (int)first,
            rows * row_bytes > kLargeTable};
    begun += Z.rows;
    const int64_t pieces = Z.ld == Z.bytes ? (Z.rows * Z.bytes + 15) / 16 : Z.rows * ((Z.bytes + 15) / 16);
    blocks = (unsigned)(first + (pieces + kZeroChunk / 16 - 1) / (kZeroChunk / 16));
    return Z;
  };
  unsigned blocks = 0;
  if (n > 0 && one) {
    const Zeros Z = zeros(1, blocks);
    hipLaunchKernelGGL(sort_one_kernel, dim3(blocks), dim3(kSortThreads), 0, s, I, (int)n, p.bits, p.passes, buf[0], Z);
  } else if (n > 0) {
    const uint2* in = nullptr;
    for (int k = 0; k < p.passes; ++k) {
      const bool scan = p.nblk > kScanBlocks;
      Zeros Z = zeros(p.nblk, blocks);
      hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(kSortThreads), 0, s, I, in, n, p.bits, k * p.bits, counts,
                         ld, Z);
      if (scan)
        hipLaunchKernelGGL(sort_scan_kernel, dim3(1u << p.bits), dim3(kSortThreads), 0, s, counts, (int)p.nblk, ld,
                           totals);
      Z = zeros(p.nblk, blocks);
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(blocks), dim3(kSortThreads), 0, s, I, in, n, p.bits, k * p.bits,
                         counts, ld, scan ? totals : nullptr, buf[k & 1], (int)p.nblk, Z);
      in = buf[k & 1];
    }
    sorted = in;
  }
  const Grad G{sorted, n, rows, dim, p.lanes_log2, p.run, p.nruns, scale, accumulate, (float*)(w + p.part), p.part_ld,
               cleared};
  if (dtype == 0) launch_sums<float>(G, dout, ldd, dtable, ldg, s);
  else if (dtype == 1) launch_sums<bf16_t>(G, dout, ldd, dtable, ldg, s);
  else launch_sums<_Float16>(G, dout, ldd, dtable, ldg, s);
  return mms::check_launch(fn);
}
