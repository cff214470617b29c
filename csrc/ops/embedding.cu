// embedding.cu - token and position embedding, and the gradients of both
// tables by sorted tokens.
//
//   y[r]  = scale w[token[r]] + p[position[r]]
//   dw[v] = scale sum over r with token[r] = v of g[r]   (likewise dp)
//
// An index outside its table contributes nothing: zero to y, and no gradient.
//
// The gradient, deterministic whatever the launch:
//   1. sortChunk     a CTA sorts 1024 to 4096 tokens with their row in the
//                    chunk. These CTAs belong to the forward pass's launch,
//                    which is bound by memory and hides most of them (65536 rows:
//                    5 us are seen of 13 as a launch of their own), and leave the
//                    sorted chunks for the backward pass;
//   2. mergeRanks    a token's place in the whole order is its place in its
//                    chunk plus the number of smaller ones in every other
//                    chunk (equal ones count in chunks before its own), found
//                    by binary searches. Not needed when a single chunk holds
//                    all rows; more than 131072 rows are merged that many
//                    at a time, then the sorted parts two and two (mergePairs),
//                    so that the work grows with rows log rows;
//   3. tableGrads    the sorted rows in blocks of 16 to 64: a group of threads,
//                    one per 16 bytes of a row, adds the gradients of each run
//                    of equal tokens in row order and writes the table row of
//                    a run that lies within its block; runs cut by a block's
//                    border leave fp32 partial sums. Other CTAs of the launch
//                    write the rows that no token names: zeros;
//   4. joinRuns      adds the partial sums of each cut run in block order.
// Without explicit positions the second table's order is known (row r has
// position r % seq) and skips the sort; both tables share the launches of 3
// and 4. Sums are fp32, rounded once to the table's type.
#include <type_traits>

#include "common.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr int kThreads = 256;

// N neighbouring values of a row. FAST: whole 8- or 16-byte pieces (cols % N
// == 0 and aligned rows); else one by one, the ones past the row's end zero.
template <int N>
struct Cols {
  float v[N];
};
// N values as they lie in memory: what a load in flight holds in registers.
template <class T, int N>
struct Raw {
  uint32_t w[N * sizeof(T) / 4];
};
template <bool FAST, int N, class T>
__device__ __forceinline__ Raw<T, N> loadRaw(const T* row, int c, int cols) {
  Raw<T, N> r;
  constexpr int W = N * sizeof(T) / 4;
  if (FAST) {
    if (W == 2) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + c));
      r.w[0] = u.x; r.w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + c) + i / 4);
        r.w[i] = u.x; r.w[i + 1] = u.y; r.w[i + 2] = u.z; r.w[i + 3] = u.w;
      }
    }
  } else if (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      r.w[i] = c + i < cols ? *reinterpret_cast<const uint32_t*>(row + c + i) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t lo = c + i < cols ? *reinterpret_cast<const uint16_t*>(row + c + i) : 0u;
      const uint32_t hi =
          c + i + 1 < cols ? *reinterpret_cast<const uint16_t*>(row + c + i + 1) : 0u;
      r.w[i / 2] = lo | hi << 16;
    }
  }
  return r;
}
template <class T, int N>
__device__ __forceinline__ Raw<T, N> zeroRaw() {
  Raw<T, N> r;
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T) / 4); ++i) r.w[i] = 0u;
  return r;
}
template <class T, int N>
__device__ __forceinline__ Cols<N> unpack(const Raw<T, N>& r) {
  Cols<N> v;
#pragma unroll
  for (int i = 0; i < N; ++i)
    v.v[i] = __uint_as_float(sizeof(T) == 4 ? r.w[i]
                             : (i & 1)      ? r.w[i / 2] & 0xffff0000u
                                            : r.w[i / 2] << 16);
  return v;
}
template <int N>
__device__ __forceinline__ void storeFast(float* p, const float* v) {
#pragma unroll
  for (int i = 0; i < N; i += 4)
    *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int N>
__device__ __forceinline__ void storeFast(uint16_t* p, const float* v) {
  const uint2 a = tobf4(make_float4(v[0], v[1], v[2], v[3]));
  if (N == 8) {
    const uint2 b = tobf4(make_float4(v[4], v[5], v[6], v[7]));
    *reinterpret_cast<uint4*>(p) = make_uint4(a.x, a.y, b.x, b.y);
  } else {
    *reinterpret_cast<uint2*>(p) = a;
  }
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = f2bf(v); }

template <bool FAST, int N, class T>
__device__ __forceinline__ Cols<N> loadCols(const T* row, int c, int cols) {
  return unpack(loadRaw<FAST, N>(row, c, cols));
}
template <bool FAST, int N, class T>
__device__ __forceinline__ void storeCols(T* row, int c, int cols, const Cols<N>& r) {
  if (FAST) {
    storeFast<N>(row + c, r.v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < cols) store1(row + c + i, r.v[i]);
  }
}
template <int N>
__device__ __forceinline__ Cols<N> zeroCols() {
  Cols<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = 0.f;
  return r;
}
template <int N>
__device__ __forceinline__ void addTo(Cols<N>& a, const Cols<N>& b) {
#pragma unroll
  for (int i = 0; i < N; ++i) a.v[i] += b.v[i];
}
template <int N>
__device__ __forceinline__ Cols<N> scaled(const Cols<N>& a, float s) {
  Cols<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = a.v[i] * s;
  return r;
}

// -- sorting ---------------------------------------------------------------------

// Sort keys are (token << bits | row in the chunk), bits = log2(chunk), so
// they differ and the order of equal tokens is the rows'. A token outside the
// table takes the value `vocab`, after all others; padding follows it.
// Keys take 32 bits where token and place in the chunk fit.
constexpr int kSmallChunk = 1024, kChunk = 2048, kLargeChunk = 4096;

template <int CHUNK>
__host__ __device__ __forceinline__ constexpr int chunkBits() {
  return CHUNK == kSmallChunk ? 10 : CHUNK == kChunk ? 11 : 12;
}

// Chunks of 1024, 2048 or 4096 rows: small ones are sorted quickly, large ones
// leave the merge fewer searches per row (one in every other chunk). Forward and
// backward pass in us (width 768, fp32 below, bf16 from 65536 rows on):
//   rows          20480   32768   65536   131072
//   chunk 1024       74      95     129      246
//   chunk 2048       78      92     120      208
//   chunk 4096        -       -     126     189
struct SortPlan {
  int chunk, chunks;
  bool wide;  // 64-bit keys
};
__host__ inline SortPlan sortPlan(int rows, int vocab) {
  SortPlan p;
  p.chunk = rows <= 24 * 1024 ? kSmallChunk : rows <= 96 * 1024 ? kChunk : kLargeChunk;
  p.chunks = (rows + p.chunk - 1) / p.chunk;
  p.wide = (int64_t)(vocab + 1ll) * p.chunk >= (1ll << 32);
  return p;
}

// What a list of indices is sorted into: the chunks' keys, or with one chunk
// the sorted indices and their rows (`second`, at the next 16 bytes).
struct SortList {
  const int64_t* index;
  void* first;
  int* second;
  int vocab, wide;
};

// The steps of a bitonic sort from (SIZE, D) on, for E neighbouring keys per
// thread: steps at a distance inside a thread's keys need no exchange, those
// inside a warp shuffle, and longer ones go through shared memory. Recursion,
// not loops: the compiler unrolls only some of the 78 steps of 4096 keys, and
// the keys then lie in memory (a forward pass of 65536 rows with chunks of 4096:
// 62 us, 51 like this).
template <int SIZE, int D, int CHUNK, int E, class Key>
__device__ __forceinline__ void sortSteps(Key (&k)[E], Key* s) {
  const int t0 = threadIdx.x * E;
  if constexpr (D < E) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (j & D) continue;
      const bool up = ((t0 + j) & SIZE) == 0;
      const Key lo = min(k[j], k[j | D]), hi = max(k[j], k[j | D]);
      k[j] = up ? lo : hi;
      k[j | D] = up ? hi : lo;
    }
  } else {
    // The partner of key i is key i ^ D, held by thread ^ (D / E).
    const bool takeMin = ((t0 & SIZE) == 0) == ((t0 & D) == 0);
    if constexpr (D >= 32 * E) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < E; ++j) s[j * kThreads + threadIdx.x] = k[j];
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < E; ++j) {
      Key other;
      if constexpr (D >= 32 * E)
        other = s[j * kThreads + (threadIdx.x ^ (D / E))];
      else
        other = __shfl_xor_sync(0xffffffffu, k[j], D / E);
      k[j] = takeMin ? min(k[j], other) : max(k[j], other);
    }
  }
  if constexpr (D > 1)
    sortSteps<SIZE, D / 2, CHUNK>(k, s);
  else if constexpr (SIZE < CHUNK)
    sortSteps<2 * SIZE, SIZE, CHUNK>(k, s);
}

// Sorts one chunk of a list, CHUNK / 256 keys per thread.
template <class Key, int CHUNK>
__device__ __noinline__ void sortChunk(const SortList& list, int rows, int chunk, bool one,
                                       Key* s) {
  constexpr int bits = chunkBits<CHUNK>();
  constexpr int E = CHUNK / kThreads;
  const int64_t* __restrict__ token = list.index;
  const int vocab = list.vocab;
  const int64_t base = (int64_t)chunk * CHUNK;
  const int t0 = threadIdx.x * E;
  Key k[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int64_t r = base + t0 + j;
    k[j] = ~(Key)0;
    if (r < rows) {
      const int64_t t = token[r];
      k[j] = ((Key)(t >= 0 && t < vocab ? t : vocab) << bits) | (Key)(t0 + j);
    }
  }
  sortSteps<2, 1, CHUNK>(k, s);
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int64_t r = base + t0 + j;
    if (r >= rows) continue;
    if (one) {
      static_cast<int*>(list.first)[r] = (int)(k[j] >> bits);
      list.second[r] = (int)(k[j] & (CHUNK - 1));
    } else {
      static_cast<Key*>(list.first)[r] = k[j];
    }
  }
}

// -- forward -----------------------------------------------------------------------

// A CTA takes `per` rows: their indices first, then the rows' pieces of N
// columns in turn, so that several loads per thread are in flight whatever the
// width. Bound by memory: a row of each table read, one written. With SORT the
// first CTAs sort the chunks of the lists.
constexpr int kFwdMaxRows = 16;
struct SortLists {
  SortList list[2];
  int lists, chunk, chunks;
};
template <class W, class Y, bool FAST, int N, bool SORT>
__global__ void __launch_bounds__(kThreads, 4)
    embeddingFwd(const int64_t* __restrict__ token, const int64_t* __restrict__ position,
                 const W* __restrict__ w, const W* __restrict__ p, Y* __restrict__ y, int rows,
                 int seq, int vocab, int context, int cols, float scale, int per,
                 const __grid_constant__ SortLists sort) {
  int cta = blockIdx.x;
  if (SORT) {
    __shared__ __align__(16) uint64_t sKeys[kLargeChunk];
    if (cta < sort.lists * sort.chunks) {
      const bool second = cta >= sort.chunks, one = sort.chunks == 1;
      const SortList& list = sort.list[second ? 1 : 0];
      const int chunk = second ? cta - sort.chunks : cta;
      auto run = [&](auto* keys) {
        using Key = std::remove_pointer_t<decltype(keys)>;
        if (sort.chunk == kSmallChunk)
          sortChunk<Key, kSmallChunk>(list, rows, chunk, one, keys);
        else if (sort.chunk == kChunk)
          sortChunk<Key, kChunk>(list, rows, chunk, one, keys);
        else
          sortChunk<Key, kLargeChunk>(list, rows, chunk, one, keys);
      };
      if (list.wide)
        run(sKeys);
      else
        run(reinterpret_cast<uint32_t*>(sKeys));
      return;
    }
    cta -= sort.lists * sort.chunks;
  }
  __shared__ const W* sW[kFwdMaxRows];
  __shared__ const W* sP[kFwdMaxRows];
  const int64_t first = (int64_t)cta * per;
  const int n = (int)min((int64_t)per, rows - first);
  if (threadIdx.x < n) {
    const int64_t r = first + threadIdx.x, t = token[r];
    const int64_t at = position ? position[r] : r % seq;
    sW[threadIdx.x] = t >= 0 && t < vocab ? w + t * cols : nullptr;
    sP[threadIdx.x] = p != nullptr && at >= 0 && at < context ? p + at * cols : nullptr;
  }
  __syncthreads();
  const uint32_t pieces = (uint32_t)(cols + N - 1) / N, all = pieces * n;
  constexpr int U = 4;
  for (uint32_t i0 = threadIdx.x; i0 < all; i0 += U * kThreads) {
    Raw<W, N> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * kThreads;
      if (i >= all) break;
      const uint32_t r = i / pieces, c = (i - r * pieces) * N;
      a[u] = sW[r] ? loadRaw<FAST, N>(sW[r], c, cols) : zeroRaw<W, N>();
      b[u] = sP[r] ? loadRaw<FAST, N>(sP[r], c, cols) : zeroRaw<W, N>();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * kThreads;
      if (i >= all) break;
      const uint32_t r = i / pieces, c = (i - r * pieces) * N;
      Cols<N> x = unpack(a[u]);
      const Cols<N> q = unpack(b[u]);
#pragma unroll
      for (int k = 0; k < N; ++k) x.v[k] = x.v[k] * scale + q.v[k];
      storeCols<FAST, N>(y + (first + r) * cols, c, cols, x);
    }
  }
}

// -- merging -----------------------------------------------------------------------

// Several chunks at a time in shared memory (128 KiB), one search in each
// going on side by side.
constexpr int kMergeThreads = 512;
constexpr uint32_t kMergeSmem = 128 * 1024;
// Rows whose chunks are merged at once. Forward and backward pass in us, bf16:
//   rows (width)    262144 (256)  524288 (256)  1048576 (256)  4194304 (64)  16777216 (4)
//   131072               214           397            771          2380         10540
//   262144               282           519           1012          3320         14370
//   1048576              282           756           2495          9230         37620
constexpr int kMergeRows = 128 * 1024;

template <class Key, int CHUNK>
__global__ void __launch_bounds__(kMergeThreads)
    mergeRanks(const Key* __restrict__ sorted, int* __restrict__ skey, int* __restrict__ perm,
               int rows) {
  extern __shared__ __align__(16) uint8_t smem[];
  Key* s = reinterpret_cast<Key*>(smem);
  constexpr int bits = chunkBits<CHUNK>();
  constexpr int at1 = kMergeSmem / (CHUNK * sizeof(Key));  // chunks at a time
  constexpr int side = 4;                                  // searches side by side
  const int64_t at = (int64_t)blockIdx.x * kMergeThreads + threadIdx.x;  // CHUNK % 512 == 0
  const int own = (int)((int64_t)blockIdx.x * kMergeThreads / CHUNK);
  constexpr int together = kMergeRows / CHUNK;
  const int chunk0 = own / together * together;
  const int chunks = min((rows + CHUNK - 1) / CHUNK, chunk0 + together);
  const int64_t end = min((int64_t)rows, (int64_t)chunks * CHUNK);
  const bool has = at < rows;
  const Key key = has ? sorted[at] : 0;
  const Key token = key >> bits;
  int rank = (int)(at - (int64_t)(own - chunk0) * CHUNK);
  for (int c0 = chunk0; c0 < chunks; c0 += at1) {
    const int64_t from = (int64_t)c0 * CHUNK;
    const int n = (int)min((int64_t)at1 * CHUNK, end - from);
    __syncthreads();
    // 16-byte pieces; the last may run past n, within the rounded-up buffer.
    for (int i = threadIdx.x; i < (int)((n * sizeof(Key) + 15) / 16); i += kMergeThreads)
      reinterpret_cast<uint4*>(smem)[i] =
          __ldg(reinterpret_cast<const uint4*>(sorted + from) + i);
    __syncthreads();
    const int here = (n + CHUNK - 1) / CHUNK;
    for (int c = 0; c < here; c += side) {
      // lo: how many of the chunk's keys come before this one.
      int lo[side], len[side];
      Key limit[side];
#pragma unroll
      for (int u = 0; u < side; ++u) {
        const int chunk = c0 + c + u;
        lo[u] = 0;
        len[u] = c + u < here && chunk != own ? min(CHUNK, n - (c + u) * CHUNK) : 0;
        limit[u] = (token + (chunk < own ? 1 : 0)) << bits;
      }
#pragma unroll 1
      for (int step = CHUNK; step > 0; step >>= 1) {
#pragma unroll
        for (int u = 0; u < side; ++u) {
          const int next = lo[u] + step;
          if (next <= len[u] && s[(c + u) * CHUNK + next - 1] < limit[u]) lo[u] = next;
        }
      }
#pragma unroll
      for (int u = 0; u < side; ++u) rank += lo[u];
    }
  }
  if (has) {
    skey[rank] = (int)token;
    perm[rank] = own * CHUNK + (int)(key & (CHUNK - 1));
  }
}

// Sorted parts of `len` places, two and two: a place's new one is its own in its
// part plus the number of smaller tokens in the other (equal ones count in the
// first part), found by a binary search. Neighbouring threads have neighbouring
// tokens, so that a warp's searches read the same few lines.
__global__ void __launch_bounds__(kThreads)
    mergePairs(const int* __restrict__ skey, const int* __restrict__ perm,
               int* __restrict__ skeyOut, int* __restrict__ permOut, int rows, int64_t len) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= rows) return;
  const int64_t part = at / len, from = min((part ^ 1) * len, (int64_t)rows);
  const int key = skey[at], limit = key + (int)(part & 1);
  int64_t lo = from, hi = min(from + len, (int64_t)rows);
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (skey[mid] < limit)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int64_t to = at - (part & 1) * len + lo - from;
  skeyOut[to] = key;
  permOut[to] = perm[at];
}

// -- gradients of the tables -------------------------------------------------------

constexpr int kMaxBlock = 64;

// A table's gradient. Sorted place i holds token key(i) of row row(i); without
// arrays the order of r % seq: place i is row (i % batch) * seq + i / batch.
struct Table {
  const int* skey;
  const int* perm;
  void* out;
  float* partial;  // [2 * blocks][cols]: a block's first run, its last run
  int seq, batch;  // used when skey is null
  int vocab;
  float scale;
  int block, blocks;  // sorted rows per block, blocks
  int sumCtas, zeroCtas;

  __device__ __forceinline__ int key(int i) const { return skey ? skey[i] : i / batch; }
  __device__ __forceinline__ int row(int i) const {
    return skey ? perm[i] : (i % batch) * seq + i / batch;
  }
};
struct TableGradArgs {
  Table table[2];
  int tables;
  int rows, cols;
  int group;  // threads per block of rows
};
constexpr int kZeroRows = 64;  // table rows per such CTA

// First place in sorted order whose key is at least v.
__device__ __forceinline__ int lowerBound(const Table& t, int rows, int v) {
  if (t.skey == nullptr) {
    const int64_t at = (int64_t)v * t.batch;
    return at < rows ? (int)at : rows;
  }
  int lo = 0, hi = rows;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.skey[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

template <class G, class W, bool FAST, int N>
__global__ void __launch_bounds__(kThreads, 4)
    tableGrads(const G* __restrict__ g, const __grid_constant__ TableGradArgs a) {
  __shared__ int sKey[kThreads / 8][kMaxBlock + 2];  // with the neighbours' keys
  __shared__ int sRow[kThreads / 8][kMaxBlock];
  __shared__ uint8_t sEmpty[kZeroRows];
  int cta = blockIdx.x, which = 0;
  // Sums of both tables first, then the rows of zeros.
  const int sums = a.table[0].sumCtas + (a.tables > 1 ? a.table[1].sumCtas : 0);
  const bool zeros = cta >= sums;
  if (zeros) cta -= sums;
  const int before = zeros ? a.table[0].zeroCtas : a.table[0].sumCtas;
  which = cta >= before;
  if (which) cta -= before;
  const Table& t = a.table[which];
  const int cols = a.cols, group = a.group;
  W* out = static_cast<W*>(t.out);
  const int tile0 = blockIdx.y * group * N;
  if (zeros) {
    // Rows without a token.
    const int v0 = cta * kZeroRows;
    if (threadIdx.x < kZeroRows) {
      const int v = v0 + threadIdx.x;
      bool empty = false;
      if (v < t.vocab) {
        const int at = lowerBound(t, a.rows, v);
        empty = at >= a.rows || t.key(at) != v;
      }
      sEmpty[threadIdx.x] = empty;
    }
    __syncthreads();
    const int c = tile0 + (threadIdx.x & (group - 1)) * N;
    if (c < cols)
      for (int i = threadIdx.x / group; i < kZeroRows; i += kThreads / group)
        if (sEmpty[i]) storeCols<FAST, N>(out + (int64_t)(v0 + i) * cols, c, cols, zeroCols<N>());
    return;
  }
  const int slot = threadIdx.x / group, lane = threadIdx.x & (group - 1);
  const int block = cta * (kThreads / group) + slot;
  const int first = block * t.block;
  const int n = min(t.block, a.rows - first);
  for (int i = lane; i < t.block + 2; i += group) {
    const int at = first + i - 1;
    sKey[slot][i] = at >= 0 && at < a.rows ? t.key(at) : -1;
    if (i >= 1 && i <= t.block && at < a.rows) sRow[slot][i - 1] = t.row(at);
  }
  __syncthreads();
  const int c = tile0 + lane * N;
  if (n <= 0 || c >= cols) return;
  const int* key = sKey[slot] + 1;
  Cols<N> acc = zeroCols<N>();
  bool head = key[0] == key[-1];  // the current run began in a block before
  constexpr int U = 8;
  for (int i0 = 0; i0 < n; i0 += U) {
    Raw<G, N> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < n) v[u] = loadRaw<FAST, N>(g + (int64_t)sRow[slot][i0 + u] * cols, c, cols);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      addTo(acc, unpack(v[u]));
      const bool ends = key[i + 1] != key[i];
      if (ends || i == n - 1) {
        if (key[i] < t.vocab) {
          if (head || !ends)
            storeCols<FAST, N>(t.partial + ((int64_t)block * 2 + (head ? 0 : 1)) * cols, c, cols,
                               acc);
          else
            storeCols<FAST, N>(out + (int64_t)key[i] * cols, c, cols, scaled(acc, t.scale));
        }
        acc = zeroCols<N>();
        head = false;
      }
    }
  }
}

// Adds the partial sums of each run that crosses a block's border, for 128
// columns (blockIdx.y). A warp looks after the run that begins in its block
// and goes on past it; a long run is added by the whole CTA, each warp an even
// share of the blocks in order.
constexpr int kJoinWarps = 16;
constexpr int kLongRun = 8;  // blocks that one warp still adds by itself

template <bool FAST>
__device__ __forceinline__ Cols<4> sumBlocks(const float* partial, int from, int to, int c,
                                             int cols) {
  Cols<4> acc = zeroCols<4>();
  constexpr int U = 4;
  for (int b0 = from; b0 < to; b0 += U) {
    Cols<4> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = b0 + u < to ? loadCols<FAST, 4>(partial + (int64_t)(b0 + u) * 2 * cols, c, cols)
                         : zeroCols<4>();
#pragma unroll
    for (int u = 0; u < U; ++u) addTo(acc, v[u]);
  }
  return acc;
}

// The first block at or past b0 whose follower does not begin with k, + 1, by
// the whole warp: each load narrows the blocks to a 33rd (65536 rows with one
// token in ten alike: the kernel takes 14.4 us, 17 with a binary search).
__device__ __forceinline__ int runEnd(const Table& t, int k, int b0) {
  const int lane = threadIdx.x & 31;
  int lo = b0, hi = t.blocks - 1;  // the block is in [lo, hi]: the last has no follower
  while (lo < hi) {
    const int step = (hi - lo + 32) / 33;
    const int b = lo + (lane + 1) * step - 1;
    const bool ends = b >= hi || t.key((b + 1) * t.block) != k;
    const uint32_t votes = __ballot_sync(0xffffffffu, ends);
    const int n = votes ? __ffs(votes) - 1 : 32;  // probes that go on
    const int from = lo + n * step;
    if (votes) hi = min(hi, from + step - 1);
    lo = min(from, hi);
  }
  return lo + 1;
}

template <class W, bool FAST>
__global__ void __launch_bounds__(kJoinWarps * 32, 3)
    joinRuns(const __grid_constant__ TableGradArgs a, int firstTable) {
  __shared__ int sLong[kJoinWarps][2];  // the token, and the last + 1 of its blocks
  __shared__ Cols<4> sPart[kJoinWarps][32];
  const Table& t = a.table[firstTable + blockIdx.z];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cols = a.cols, c = blockIdx.y * 128 + lane * 4;
  const int block = blockIdx.x * kJoinWarps + warp;
  const int first = block * t.block, last = min(first + t.block, a.rows) - 1;
  W* out = static_cast<W*>(t.out);
  int token = -1, end = 0;  // blocks block + 1 .. end - 1 go on with the run
  if (block < t.blocks && last + 1 < a.rows) {
    // The keys that decide, one per lane: this block's ends and neighbours.
    const int at = lane == 0 ? last : lane == 1 ? last + 1 : lane == 2 ? first : first - 1;
    const int k4 = lane < 4 && at >= 0 ? t.key(at) : -1;
    const int k = __shfl_sync(0xffffffffu, k4, 0), after = __shfl_sync(0xffffffffu, k4, 1);
    const int begin = __shfl_sync(0xffffffffu, k4, 2), before = __shfl_sync(0xffffffffu, k4, 3);
    if (k == after && k < t.vocab && (begin != k || before != k)) {
      token = k;
      // The run ends with the first of the next 32 blocks whose follower
      // does not begin with the token; past them, a search.
      const int b = block + 1 + lane;
      const bool ends = b >= t.blocks - 1 || t.key((b + 1) * t.block) != k;
      const uint32_t votes = __ballot_sync(0xffffffffu, ends);
      end = votes ? block + 1 + __ffs(votes) : runEnd(t, k, block + 33);
    }
  }
  const bool isLong = token >= 0 && end - block > kLongRun;
  if (token >= 0 && !isLong && c < cols) {
    Cols<4> sum = loadCols<FAST, 4>(t.partial + ((int64_t)block * 2 + 1) * cols, c, cols);
    addTo(sum, sumBlocks<FAST>(t.partial, block + 1, end, c, cols));
    storeCols<FAST, 4>(out + (int64_t)token * cols, c, cols, scaled(sum, t.scale));
  }
  if (lane == 0) {
    sLong[warp][0] = isLong ? token : -1;
    sLong[warp][1] = end;
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    if (sLong[w][0] < 0) continue;  // the same for the whole CTA
    const int from = blockIdx.x * kJoinWarps + w + 1, to = sLong[w][1];
    const int per = (to - from + kJoinWarps - 1) / kJoinWarps;
    if (c < cols)
      sPart[warp][lane] = sumBlocks<FAST>(t.partial, min(to, from + warp * per),
                                          min(to, from + (warp + 1) * per), c, cols);
    __syncthreads();
    if (warp == 0 && c < cols) {
      Cols<4> sum = loadCols<FAST, 4>(t.partial + ((int64_t)(from - 1) * 2 + 1) * cols, c, cols);
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) addTo(sum, sPart[i][lane]);
      storeCols<FAST, 4>(out + (int64_t)sLong[w][0] * cols, c, cols, scaled(sum, t.scale));
    }
    __syncthreads();
  }
}

// -- launches ----------------------------------------------------------------------

// The least power of two from 8 to 64 that covers cols with n columns per
// thread.
int groupFor(int cols, int n) {
  int g = 8;
  while (g < 64 && g * n < cols) g *= 2;
  return g;
}
// Whether rows of `cols` values from p on divide into aligned pieces of n.
bool pieces(const void* p, int valueBytes, int cols, int n) {
  const uintptr_t bytes = (uintptr_t)(n * valueBytes < 16 ? n * valueBytes : 16);
  return p == nullptr || (cols % n == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0);
}

template <class W, class Y>
int fwd(const int64_t* token, const int64_t* position, const void* w, const void* p, void* y,
        int rows, int seq, int vocab, int context, int cols, float scale, const SortLists& sort,
        cudaStream_t stream) {
  constexpr int N = 16 / sizeof(W);  // 16-byte loads
  const bool fast = pieces(w, sizeof(W), cols, N) && pieces(p, sizeof(W), cols, N) &&
                    pieces(y, sizeof(Y), cols, N);
  // Few rows spread over the SMs; many take 16 to a CTA.
  int per = (rows + kSMs * 4 - 1) / (kSMs * 4);
  if (per > kFwdMaxRows) per = kFwdMaxRows;
  auto kernel = sort.lists == 0 ? (fast ? embeddingFwd<W, Y, true, N, false>
                                        : embeddingFwd<W, Y, false, 4, false>)
                                : (fast ? embeddingFwd<W, Y, true, N, true>
                                        : embeddingFwd<W, Y, false, 4, true>);
  const unsigned ctas = (unsigned)((rows + per - 1) / per) + (unsigned)(sort.lists * sort.chunks);
  kernel<<<ctas, kThreads, 0, stream>>>(token, position, static_cast<const W*>(w),
                                        static_cast<const W*>(p), static_cast<Y*>(y), rows, seq,
                                        vocab, context, cols, scale, per, sort);
  return launched(cudaGetLastError());
}

template <class Key, int CHUNK>
int mergeChunks(const void* sorted, int* skey, int* perm, int rows, int chunks,
                cudaStream_t stream) {
  auto merge = mergeRanks<Key, CHUNK>;
  static std::atomic<uint64_t> done{0};  // devices (bit d) with the shared memory opted in
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 3;
  if (!(done.load(std::memory_order_acquire) & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(
        merge, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMergeSmem);
    if (e != cudaSuccess) return (int)e;
    done.fetch_or(1ull << dev, std::memory_order_acq_rel);
  }
  const uint64_t bytes = (uint64_t)chunks * CHUNK * sizeof(Key);
  merge<<<(rows + kMergeThreads - 1) / kMergeThreads, kMergeThreads,
          bytes < kMergeSmem ? bytes : kMergeSmem, stream>>>(static_cast<const Key*>(sorted), skey,
                                                            perm, rows);
  return launched(cudaGetLastError());
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
// Two lists, sorted tokens and their rows; a pass of mergePairs needs two more.
size_t listsBytes(int64_t rows) { return 2 * round16(4 * rows); }
size_t sortBytes(int64_t rows) { return (rows > kMergeRows ? 2 : 1) * listsBytes(rows); }

// Sorts whole from sorted chunks; lists in `at`, sortBytes(rows) of scratch.
int mergeChunks(const SortPlan& p, const void* sorted, char* at, int rows, const int** skey,
                const int** perm, cudaStream_t stream) {
  auto pick = [&](auto key) {
    using Key = decltype(key);
    return p.chunk == kSmallChunk ? mergeChunks<Key, kSmallChunk>
           : p.chunk == kChunk    ? mergeChunks<Key, kChunk>
                                  : mergeChunks<Key, kLargeChunk>;
  };
  auto f = p.wide ? pick(uint64_t{}) : pick(uint32_t{});
  auto lists = [&](bool second, int** k, int** r) {
    char* base = at + (second ? listsBytes(rows) : 0);
    *k = reinterpret_cast<int*>(base);
    *r = reinterpret_cast<int*>(base + listsBytes(rows) / 2);
  };
  int *k, *r, *k2, *r2;
  bool second = false;
  lists(second, &k, &r);
  if (int rc = f(sorted, k, r, rows, p.chunks, stream)) return rc;
  for (int64_t len = kMergeRows; len < rows; len *= 2) {
    second = !second;
    lists(second, &k2, &r2);
    mergePairs<<<(unsigned)(((int64_t)rows + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
        k, r, k2, r2, rows, len);
    if (int rc = launched(cudaGetLastError())) return rc;
    k = k2;
    r = r2;
  }
  *skey = k;
  *perm = r;
  return 0;
}

// Sorted rows per block: 16, or 32 where there are many rows (half the partial
// sums; fewer rows would leave SMs idle). Where every run has `batch` rows,
// whole runs, as long as they fit.
int blockRows(int rows, int batch) {
  if (batch > 0 && batch <= kMaxBlock) return batch <= 16 ? 16 / batch * batch : batch;
  return rows > 16 * kSmallChunk ? 32 : 16;
}

template <class G, class W>
int tableGradients(const void* g, const TableGradArgs& args, cudaStream_t stream) {
  TableGradArgs a = args;
  constexpr int N = 16 / sizeof(G);  // 16-byte loads
  bool fast = pieces(g, sizeof(G), a.cols, N), fast4 = true;
  for (int i = 0; i < a.tables; ++i) {
    fast = fast && pieces(a.table[i].out, sizeof(W), a.cols, N);
    fast4 = fast4 && pieces(a.table[i].out, sizeof(W), a.cols, 4);
  }
  const int n = fast ? N : 4;
  a.group = groupFor(a.cols, n);
  const int perCta = kThreads / a.group;
  int ctas = 0, joinFrom = a.tables, joinBlocks = 0;
  for (int i = 0; i < a.tables; ++i) {
    Table& t = a.table[i];
    t.block = blockRows(a.rows, t.skey ? 0 : t.batch);
    t.blocks = (a.rows + t.block - 1) / t.block;
    t.sumCtas = (t.blocks + perCta - 1) / perCta;
    t.zeroCtas = (t.vocab + kZeroRows - 1) / kZeroRows;
    ctas += t.sumCtas + t.zeroCtas;
    // Blocks of whole runs have nothing to join.
    if (t.blocks == 1 || (!t.skey && t.block % t.batch == 0)) continue;
    if (joinFrom == a.tables) joinFrom = i;
    if (t.blocks > joinBlocks) joinBlocks = t.blocks;
  }
  const unsigned tiles = (unsigned)((a.cols + a.group * n - 1) / (a.group * n));
  auto sum = fast ? tableGrads<G, W, true, N> : tableGrads<G, W, false, 4>;
  sum<<<dim3((unsigned)ctas, tiles), kThreads, 0, stream>>>(static_cast<const G*>(g), a);
  if (int rc = launched(cudaGetLastError())) return rc;
  if (joinFrom == a.tables) return 0;
  // Tables joinFrom ... up to the last that has something to join: the first
  // alone unless the second has too.
  const Table& last = a.table[a.tables - 1];
  const bool second = a.tables > 1 && joinFrom == 0 && last.blocks > 1 &&
                      (last.skey || last.block % last.batch != 0);
  auto join = fast4 ? joinRuns<W, true> : joinRuns<W, false>;
  join<<<dim3((unsigned)((joinBlocks + kJoinWarps - 1) / kJoinWarps),
              (unsigned)((a.cols + 127) / 128), second ? 2u : 1u),
         kJoinWarps * 32, 0, stream>>>(a, joinFrom);
  return launched(cudaGetLastError());
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
constexpr int64_t kMostRows = INT32_MAX - kLargeChunk;

// Scratch of one table beside its sortBytes.
size_t partialBytes(int64_t rows, int cols) {
  return round16(sizeof(float) * 2 * ((rows + 15) / 16) * cols);
}

}  // namespace
}  // namespace tnops

using namespace tnops;

extern "C" size_t tnops_embedding_order_bytes(int64_t rows, int size) {
  if (rows <= 0 || rows > kMostRows || size <= 0 || size == INT32_MAX) return 0;
  const SortPlan p = sortPlan((int)rows, size);
  return p.chunks == 1 ? 2 * round16(4 * rows) : round16((p.wide ? 8 : 4) * rows);
}

extern "C" int tnops_embedding_fwd(const int64_t* token, const int64_t* position, const void* w,
                                   const void* p, int w_f32, void* y, int y_f32, int64_t rows,
                                   int seq, int vocab, int context, int cols, float scale,
                                   void* token_order, void* position_order, cudaStream_t stream) {
  if (rows <= 0 || rows > kMostRows || seq <= 0 || vocab <= 0 || cols <= 0 ||
      (p && context <= 0) || (token_order && vocab == INT32_MAX) || !aligned16(token_order) ||
      (position_order && (!position || context <= 0 || context == INT32_MAX)) ||
      !aligned16(position_order))
    return 1;
  SortLists sort{};
  auto add = [&](const int64_t* index, void* order, int size) {
    if (order == nullptr) return;
    const SortPlan plan = sortPlan((int)rows, size);
    sort.chunk = plan.chunk;
    sort.chunks = plan.chunks;
    sort.list[sort.lists++] = {
        index, order, reinterpret_cast<int*>(static_cast<char*>(order) + round16(4 * rows)), size,
        plan.wide};
  };
  add(token, token_order, vocab);
  add(position, position_order, context);
  auto f = w_f32 ? (y_f32 ? fwd<float, float> : fwd<float, uint16_t>)
                 : (y_f32 ? fwd<uint16_t, float> : fwd<uint16_t, uint16_t>);
  return f(token, position, w, p, y, (int)rows, seq, vocab, context, cols, scale, sort, stream);
}

extern "C" size_t tnops_embedding_grad_scratch(int64_t rows, int cols, int tables) {
  return rows <= 0 || cols <= 0 ? 0 : tables * (sortBytes(rows) + partialBytes(rows, cols));
}

extern "C" int tnops_embedding_grad(const void* g, int g_f32, const void* token_order, void* dw,
                                    int vocab, float scale, const void* position_order, int seq,
                                    void* dp, int context, int d_f32, int64_t rows, int cols,
                                    void* scratch, cudaStream_t stream) {
  if (rows <= 0 || rows > kMostRows || cols <= 0 || (!dw && !dp) ||
      (dw && (!token_order || vocab <= 0 || vocab == INT32_MAX)) || !aligned16(token_order) ||
      (dp && (context <= 0 || context == INT32_MAX ||
              (!position_order && (seq <= 0 || rows % seq)))) ||
      !aligned16(position_order) || scratch == nullptr || !aligned16(scratch))
    return 1;
  TableGradArgs a{};
  a.rows = (int)rows;
  a.cols = cols;
  char* at = static_cast<char*>(scratch);
  auto add = [&](const void* order, void* out, int n, float s) {
    Table& t = a.table[a.tables++];
    t.out = out;
    t.vocab = n;
    t.scale = s;
    t.seq = seq;
    t.batch = order ? 1 : (int)(rows / seq);
    t.partial = reinterpret_cast<float*>(at);
    at += partialBytes(rows, cols);
    if (order == nullptr) return 0;
    const SortPlan plan = sortPlan((int)rows, n);
    if (plan.chunks == 1) {
      t.skey = static_cast<const int*>(order);
      t.perm = reinterpret_cast<const int*>(static_cast<const char*>(order) + round16(4 * rows));
      return 0;
    }
    char* lists = at;
    at += sortBytes(rows);
    return mergeChunks(plan, order, lists, (int)rows, &t.skey, &t.perm, stream);
  };
  if (dw)
    if (int rc = add(token_order, dw, vocab, scale)) return rc;
  if (dp)
    if (int rc = add(position_order, dp, context, 1.0f)) return rc;
  auto f = g_f32 ? (d_f32 ? tableGradients<float, float> : tableGradients<float, uint16_t>)
                 : (d_f32 ? tableGradients<uint16_t, float> : tableGradients<uint16_t, uint16_t>);
  return f(g, a, stream);
}
