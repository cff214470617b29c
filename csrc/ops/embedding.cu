// embedding.cu - token and position embedding, and the gradients of both
// tables by sorted tokens.
//
//   y[r]  = scale w[token[r]] + p[position[r]]
//   dw[v] = scale sum over r with token[r] = v of g[r]   (likewise dp)
//
// An index outside its table contributes nothing: zero to y, and no gradient.
//
// The gradient, deterministic whatever the launch:
//   1. sortChunks    a CTA sorts 1024 (or 4096) tokens with their row in the
//                    chunk in shared memory;
//   2. mergeRanks    a token's place in the whole order is its place in its
//                    chunk plus the number of smaller ones in every other
//                    chunk (equal ones count in chunks before its own), found
//                    by binary searches: a stable sort in two launches, one
//                    when a single chunk holds all rows;
//   3. tableGrads    the sorted rows in blocks of 16: a group of threads, one
//                    per four columns, adds the gradients of each run of
//                    equal tokens in row order and writes the table row of a
//                    run that lies within its block; runs cut by a block's
//                    border leave fp32 partial sums. Other CTAs of the launch
//                    write the rows that no token names: zeros;
//   4. joinRuns      adds the partial sums of each cut run in block order.
// Without explicit positions the second table's order is known (row r has
// position r % seq) and skips the sort; both tables share the launches of 3
// and 4. Sums are fp32, rounded once to the table's type.
#include "common.cuh"
#include "tnccl_ops.h"

namespace tnops {
namespace {

constexpr int kThreads = 256;

// Four neighbouring values.
__device__ __forceinline__ float4 load4(const float* p) {
  return __ldg(reinterpret_cast<const float4*>(p));
}
__device__ __forceinline__ float4 load4(const uint16_t* p) {
  return bf4(__ldg(reinterpret_cast<const uint2*>(p)));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(uint16_t* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = tobf4(v);
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = f2bf(v); }

// Columns c .. c + 3 of a row of `cols`: whole when VEC (cols % 4 == 0 and
// aligned rows), else one by one with the missing ones zero.
template <bool VEC, class T>
__device__ __forceinline__ float4 loadCols(const T* row, int c, int cols) {
  if (VEC) return load4(row + c);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  v.x = load1(row + c);
  if (c + 1 < cols) v.y = load1(row + c + 1);
  if (c + 2 < cols) v.z = load1(row + c + 2);
  if (c + 3 < cols) v.w = load1(row + c + 3);
  return v;
}
template <bool VEC, class T>
__device__ __forceinline__ void storeCols(T* row, int c, int cols, float4 v) {
  if (VEC) {
    store4(row + c, v);
    return;
  }
  store1(row + c, v.x);
  if (c + 1 < cols) store1(row + c + 1, v.y);
  if (c + 2 < cols) store1(row + c + 2, v.z);
  if (c + 3 < cols) store1(row + c + 3, v.w);
}
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float4 scale4(float4 a, float s) {
  return make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
}

// A group of `group` threads (a power of two) per row, four columns each and
// `group * 4` apart, several rows in flight per group. Bound by memory: a row
// of each table read, one written.
constexpr int kFwdRows = 4;
template <class W, class Y, bool VEC>
__global__ void __launch_bounds__(kThreads)
    embeddingFwd(const int64_t* __restrict__ token, const int64_t* __restrict__ position,
                 const W* __restrict__ w, const W* __restrict__ p, Y* __restrict__ y, int rows,
                 int seq, int vocab, int context, int cols, float scale, int group) {
  const int lane = threadIdx.x & (group - 1);
  const int64_t first =
      ((int64_t)blockIdx.x * (kThreads / group) + threadIdx.x / group) * kFwdRows;
  const W* wr[kFwdRows];
  const W* pr[kFwdRows];
#pragma unroll
  for (int i = 0; i < kFwdRows; ++i) {
    wr[i] = pr[i] = nullptr;
    const int64_t r = first + i;
    if (r >= rows) continue;
    const int64_t t = token[r], at = position ? position[r] : r % seq;
    if (t >= 0 && t < vocab) wr[i] = w + t * cols;
    if (p != nullptr && at >= 0 && at < context) pr[i] = p + at * cols;
  }
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = lane * 4; c < cols; c += group * 4) {
    float4 a[kFwdRows], b[kFwdRows];
#pragma unroll
    for (int i = 0; i < kFwdRows; ++i) {
      a[i] = wr[i] ? loadCols<VEC>(wr[i], c, cols) : zero;
      b[i] = pr[i] ? loadCols<VEC>(pr[i], c, cols) : zero;
    }
#pragma unroll
    for (int i = 0; i < kFwdRows; ++i)
      if (first + i < rows)
        storeCols<VEC>(y + (first + i) * cols, c, cols,
                       make_float4(a[i].x * scale + b[i].x, a[i].y * scale + b[i].y,
                                   a[i].z * scale + b[i].z, a[i].w * scale + b[i].w));
  }
}

// -- sorting ---------------------------------------------------------------------

// Sort keys are (token << bits | row in the chunk), bits = log2(chunk), so
// they differ and the order of equal tokens is the rows'. A token outside the
// table takes the value `vocab`, after all others; padding follows it.
constexpr int kSmallChunk = 1024, kLargeChunk = 4096;
constexpr int kSortThreads = 1024;

template <class Key, int CHUNK>
__device__ __forceinline__ constexpr int chunkBits() {
  return CHUNK == 1024 ? 10 : 12;
}

// Bitonic sort of CHUNK keys. A thread holds pairs only in shared memory; the
// steps at distances below 32 pairs need no more than warp order, but a CTA
// barrier each keeps this short kernel simple. With one chunk the result
// goes straight to `skey` / `perm`.
template <class Key, int CHUNK>
__global__ void __launch_bounds__(kSortThreads)
    sortChunks(const int64_t* __restrict__ token, Key* __restrict__ sorted,
               int* __restrict__ skey, int* __restrict__ perm, int rows, int vocab) {
  __shared__ Key s[CHUNK];
  constexpr int bits = chunkBits<Key, CHUNK>();
  const int64_t base = (int64_t)blockIdx.x * CHUNK;
  for (int i = threadIdx.x; i < CHUNK; i += kSortThreads) {
    Key k = ~(Key)0;
    if (base + i < rows) {
      const int64_t t = token[base + i];
      k = ((Key)(t >= 0 && t < vocab ? t : vocab) << bits) | (Key)i;
    }
    s[i] = k;
  }
  __syncthreads();
  for (int size = 2; size <= CHUNK; size <<= 1)
    for (int d = size >> 1; d > 0; d >>= 1) {
      for (int t = threadIdx.x; t < CHUNK / 2; t += kSortThreads) {
        const int i = 2 * t - (t & (d - 1)), j = i + d;
        const Key a = s[i], b = s[j];
        if ((a > b) == ((i & size) == 0)) {
          s[i] = b;
          s[j] = a;
        }
      }
      __syncthreads();
    }
  for (int i = threadIdx.x; i < CHUNK && base + i < rows; i += kSortThreads) {
    const Key k = s[i];
    if (gridDim.x == 1) {
      skey[i] = (int)(k >> bits);
      perm[i] = (int)(k & (CHUNK - 1));
    } else {
      sorted[base + i] = k;
    }
  }
}

constexpr int kMergeThreads = 512;

template <class Key, int CHUNK>
__global__ void __launch_bounds__(kMergeThreads)
    mergeRanks(const Key* __restrict__ sorted, int* __restrict__ skey, int* __restrict__ perm,
               int rows) {
  __shared__ Key s[CHUNK];
  constexpr int bits = chunkBits<Key, CHUNK>();
  const int64_t at = (int64_t)blockIdx.x * kMergeThreads + threadIdx.x;  // CHUNK % 512 == 0
  const int own = (int)((int64_t)blockIdx.x * kMergeThreads / CHUNK);
  const int chunks = (rows + CHUNK - 1) / CHUNK;
  const bool has = at < rows;
  const Key key = has ? sorted[at] : 0;
  const Key token = key >> bits;
  int rank = (int)(at - (int64_t)own * CHUNK);
  for (int c = 0; c < chunks; ++c) {
    if (c == own) continue;
    const int n = min(CHUNK, rows - c * CHUNK);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kMergeThreads) s[i] = sorted[(int64_t)c * CHUNK + i];
    __syncthreads();
    // The keys below `limit` come before this one.
    const Key limit = (token + (c < own ? 1 : 0)) << bits;
    int lo = 0;
#pragma unroll
    for (int step = CHUNK; step > 0; step >>= 1)
      if (lo + step <= n && s[lo + step - 1] < limit) lo += step;
    rank += lo;
  }
  if (has) {
    skey[rank] = (int)token;
    perm[rank] = own * CHUNK + (int)(key & (CHUNK - 1));
  }
}

// -- gradients of the tables -------------------------------------------------------

constexpr int kBlock = 16;  // sorted rows per block

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

  __device__ __forceinline__ int key(int i) const { return skey ? skey[i] : i / batch; }
  __device__ __forceinline__ int row(int i) const {
    return skey ? perm[i] : (i % batch) * seq + i / batch;
  }
};
struct TableGradArgs {
  Table table[2];
  int tables;
  int rows, cols;
  int blocks;           // ceil(rows / kBlock)
  int group, sumCtas;   // threads per block of rows, CTAs of them per table
  int zeroCtas[2];      // CTAs that write rows without a token
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

template <class G, class W, bool VEC>
__global__ void __launch_bounds__(kThreads)
    tableGrads(const G* __restrict__ g, const __grid_constant__ TableGradArgs a) {
  __shared__ int sKey[kThreads / 8][kBlock + 2];  // with the neighbours' keys
  __shared__ int sRow[kThreads / 8][kBlock];
  __shared__ uint8_t sEmpty[kZeroRows];
  int cta = blockIdx.x, which = 0;
  if (cta >= a.sumCtas + a.zeroCtas[0]) {
    cta -= a.sumCtas + a.zeroCtas[0];
    which = 1;
  }
  const Table& t = a.table[which];
  const int cols = a.cols, group = a.group;
  W* out = static_cast<W*>(t.out);
  const int tile0 = blockIdx.y * group * 4;
  if (cta >= a.sumCtas) {
    // Rows without a token.
    const int v0 = (cta - a.sumCtas) * kZeroRows;
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
    const int c = tile0 + (threadIdx.x & (group - 1)) * 4;
    if (c < cols)
      for (int i = threadIdx.x / group; i < kZeroRows; i += kThreads / group)
        if (sEmpty[i])
          storeCols<VEC>(out + (int64_t)(v0 + i) * cols, c, cols,
                         make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int slot = threadIdx.x / group, lane = threadIdx.x & (group - 1);
  const int block = cta * (kThreads / group) + slot;
  const int first = block * kBlock;
  const int n = min(kBlock, a.rows - first);
  for (int i = lane; i < kBlock + 2; i += group) {
    const int at = first + i - 1;
    sKey[slot][i] = at >= 0 && at < a.rows ? t.key(at) : -1;
    if (i >= 1 && i <= kBlock && at < a.rows) sRow[slot][i - 1] = t.row(at);
  }
  __syncthreads();
  const int c = tile0 + lane * 4;
  if (n <= 0 || c >= cols) return;
  const int* key = sKey[slot] + 1;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  bool head = key[0] == key[-1];  // the current run began in a block before
  constexpr int U = 8;
  for (int i0 = 0; i0 < n; i0 += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u < n) v[u] = loadCols<VEC>(g + (int64_t)sRow[slot][i0 + u] * cols, c, cols);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= n) break;
      acc = add4(acc, v[u]);
      const bool ends = key[i + 1] != key[i];
      if (ends || i == n - 1) {
        if (key[i] < t.vocab) {
          if (head || !ends)
            storeCols<VEC>(t.partial + ((int64_t)block * 2 + (head ? 0 : 1)) * cols, c, cols, acc);
          else
            storeCols<VEC>(out + (int64_t)key[i] * cols, c, cols, scale4(acc, t.scale));
        }
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
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
constexpr int kLongRun = 32;  // blocks that one warp still adds by itself

template <bool VEC>
__device__ __forceinline__ float4 sumBlocks(const float* partial, int from, int to, int c,
                                            int cols) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 8;
  for (int b0 = from; b0 < to; b0 += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = b0 + u < to ? loadCols<VEC>(partial + (int64_t)(b0 + u) * 2 * cols, c, cols)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) acc = add4(acc, v[u]);
  }
  return acc;
}

template <class W, bool VEC>
__global__ void __launch_bounds__(kJoinWarps * 32)
    joinRuns(const __grid_constant__ TableGradArgs a) {
  __shared__ int sLong[kJoinWarps][2];  // first and last + 1 of its later blocks
  __shared__ float4 sPart[kJoinWarps][32];
  const Table& t = a.table[blockIdx.z];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cols = a.cols, c = blockIdx.y * 128 + lane * 4;
  const int block = blockIdx.x * kJoinWarps + warp;
  const int first = block * kBlock, last = min(first + kBlock, a.rows) - 1;
  W* out = static_cast<W*>(t.out);
  int token = -1, end = 0;  // blocks block + 1 .. end - 1 go on with the run
  if (block < a.blocks && last + 1 < a.rows) {
    const int k = t.key(last);
    const bool begins = t.key(first) != k || first == 0 || t.key(first - 1) != k;
    if (begins && k < t.vocab && t.key(last + 1) == k) {
      token = k;
      end = (lowerBound(t, a.rows, k + 1) - 1) / kBlock + 1;
    }
  }
  const bool isLong = token >= 0 && end - block > kLongRun;
  if (token >= 0 && !isLong && c < cols) {
    const float4 head = loadCols<VEC>(t.partial + ((int64_t)block * 2 + 1) * cols, c, cols);
    const float4 rest = sumBlocks<VEC>(t.partial, block + 1, end, c, cols);
    storeCols<VEC>(out + (int64_t)token * cols, c, cols, scale4(add4(head, rest), t.scale));
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
      sPart[warp][lane] = sumBlocks<VEC>(t.partial, min(to, from + warp * per),
                                         min(to, from + (warp + 1) * per), c, cols);
    __syncthreads();
    if (warp == 0 && c < cols) {
      float4 acc = loadCols<VEC>(t.partial + ((int64_t)(from - 1) * 2 + 1) * cols, c, cols);
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) acc = add4(acc, sPart[i][lane]);
      storeCols<VEC>(out + (int64_t)sLong[w][0] * cols, c, cols, scale4(acc, t.scale));
    }
    __syncthreads();
  }
}

// -- launches ----------------------------------------------------------------------

// The least power of two from 8 to `most` that covers cols with four columns
// per thread.
int groupFor(int cols, int most) {
  int g = 8;
  while (g < most && g * 4 < cols) g *= 2;
  return g;
}
bool vectorRows(int cols, std::initializer_list<const void*> fp32,
                std::initializer_list<const void*> bf16) {
  if (cols % 4 != 0) return false;
  uintptr_t bits = 0, bits2 = 0;
  for (const void* p : fp32) bits |= reinterpret_cast<uintptr_t>(p);
  for (const void* p : bf16) bits2 |= reinterpret_cast<uintptr_t>(p);
  return (bits & 15) == 0 && (bits2 & 7) == 0;
}

template <class W, class Y>
int fwd(const int64_t* token, const int64_t* position, const void* w, const void* p, void* y,
        int rows, int seq, int vocab, int context, int cols, float scale, cudaStream_t stream) {
  const bool wF32 = sizeof(W) == 4, yF32 = sizeof(Y) == 4;
  const bool vec = vectorRows(cols, {wF32 ? w : nullptr, wF32 ? p : nullptr, yF32 ? y : nullptr},
                              {wF32 ? nullptr : w, wF32 ? nullptr : p, yF32 ? nullptr : y});
  const int group = groupFor(cols, kThreads);
  const int64_t perCta = (int64_t)(kThreads / group) * kFwdRows;
  auto kernel = vec ? embeddingFwd<W, Y, true> : embeddingFwd<W, Y, false>;
  kernel<<<(unsigned)((rows + perCta - 1) / perCta), kThreads, 0, stream>>>(
      token, position, static_cast<const W*>(w), static_cast<const W*>(p), static_cast<Y*>(y),
      rows, seq, vocab, context, cols, scale, group);
  return launched(cudaGetLastError());
}

template <class Key, int CHUNK>
int sortTokens(const int64_t* token, void* sorted, int* skey, int* perm, int rows, int vocab,
               cudaStream_t stream) {
  const int chunks = (rows + CHUNK - 1) / CHUNK;
  sortChunks<Key, CHUNK><<<chunks, kSortThreads, 0, stream>>>(token, static_cast<Key*>(sorted),
                                                              skey, perm, rows, vocab);
  if (int rc = launched(cudaGetLastError())) return rc;
  if (chunks == 1) return 0;
  mergeRanks<Key, CHUNK><<<(rows + kMergeThreads - 1) / kMergeThreads, kMergeThreads, 0, stream>>>(
      static_cast<const Key*>(sorted), skey, perm, rows);
  return launched(cudaGetLastError());
}
// Chunks of 1024 up to 16384 rows (the sort's one CTA per chunk is what takes
// the time), of 4096 above (there each row's searches do, one per chunk). Keys
// take 32 bits where token and place in the chunk fit.
int sortTokens(const int64_t* token, void* sorted, int* skey, int* perm, int rows, int vocab,
               cudaStream_t stream) {
  if (rows <= 16 * kSmallChunk) {
    if (vocab < (1 << 22) - 1)
      return sortTokens<uint32_t, kSmallChunk>(token, sorted, skey, perm, rows, vocab, stream);
    return sortTokens<uint64_t, kSmallChunk>(token, sorted, skey, perm, rows, vocab, stream);
  }
  if (vocab < (1 << 20) - 1)
    return sortTokens<uint32_t, kLargeChunk>(token, sorted, skey, perm, rows, vocab, stream);
  return sortTokens<uint64_t, kLargeChunk>(token, sorted, skey, perm, rows, vocab, stream);
}

template <class G, class W>
int tableGradients(const void* g, const TableGradArgs& args, cudaStream_t stream) {
  TableGradArgs a = args;
  const bool gF32 = sizeof(G) == 4, wF32 = sizeof(W) == 4;
  const void* o0 = a.table[0].out;
  const void* o1 = a.tables > 1 ? a.table[1].out : nullptr;
  const bool vec =
      vectorRows(a.cols,
                 {gF32 ? g : nullptr, wF32 ? o0 : nullptr, wF32 ? o1 : nullptr,
                  a.table[0].partial, a.tables > 1 ? a.table[1].partial : nullptr},
                 {gF32 ? nullptr : g, wF32 ? nullptr : o0, wF32 ? nullptr : o1});
  a.group = groupFor(a.cols, 64);
  a.blocks = (a.rows + kBlock - 1) / kBlock;
  const int perCta = kThreads / a.group;
  a.sumCtas = (a.blocks + perCta - 1) / perCta;
  int ctas = 0;
  for (int i = 0; i < a.tables; ++i) {
    a.zeroCtas[i] = (a.table[i].vocab + kZeroRows - 1) / kZeroRows;
    ctas += a.sumCtas + a.zeroCtas[i];
  }
  const unsigned tiles = (unsigned)((a.cols + a.group * 4 - 1) / (a.group * 4));
  auto sum = vec ? tableGrads<G, W, true> : tableGrads<G, W, false>;
  sum<<<dim3((unsigned)ctas, tiles), kThreads, 0, stream>>>(static_cast<const G*>(g), a);
  if (int rc = launched(cudaGetLastError())) return rc;
  if (a.blocks == 1) return 0;  // no border to cross
  auto join = vec ? joinRuns<W, true> : joinRuns<W, false>;
  join<<<dim3((unsigned)((a.blocks + kJoinWarps - 1) / kJoinWarps),
              (unsigned)((a.cols + 127) / 128), (unsigned)a.tables),
         kJoinWarps * 32, 0, stream>>>(a);
  return launched(cudaGetLastError());
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
// Scratch of one table: sort keys, sorted keys and rows, partial sums.
size_t sortBytes(int64_t rows) { return round16(8 * rows) + 2 * round16(4 * rows); }
size_t partialBytes(int64_t rows, int cols) {
  return round16(sizeof(float) * 2 * ((rows + kBlock - 1) / kBlock) * cols);
}

}  // namespace
}  // namespace tnops

using namespace tnops;

extern "C" int tnops_embedding_fwd(const int64_t* token, const int64_t* position, const void* w,
                                   const void* p, int w_f32, void* y, int y_f32, int64_t rows,
                                   int seq, int vocab, int context, int cols, float scale,
                                   cudaStream_t stream) {
  if (rows <= 0 || rows > INT32_MAX || seq <= 0 || vocab <= 0 || cols <= 0 || (p && context <= 0))
    return 1;
  auto f = w_f32 ? (y_f32 ? fwd<float, float> : fwd<float, uint16_t>)
                 : (y_f32 ? fwd<uint16_t, float> : fwd<uint16_t, uint16_t>);
  return f(token, position, w, p, y, (int)rows, seq, vocab, context, cols, scale, stream);
}

extern "C" size_t tnops_embedding_grad_scratch(int64_t rows, int cols, int tables) {
  return rows <= 0 || cols <= 0 ? 0 : tables * (sortBytes(rows) + partialBytes(rows, cols));
}

extern "C" int tnops_embedding_grad(const void* g, int g_f32, const int64_t* token, void* dw,
                                    int vocab, float scale, const int64_t* position, int seq,
                                    void* dp, int context, int d_f32, int64_t rows, int cols,
                                    void* scratch, cudaStream_t stream) {
  if (rows <= 0 || rows > INT32_MAX - kLargeChunk || cols <= 0 || (!dw && !dp) ||
      (dw && (!token || vocab <= 0 || vocab == INT32_MAX)) ||
      (dp && (context <= 0 || context == INT32_MAX || (!position && (seq <= 0 || rows % seq)))) ||
      scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15))
    return 1;
  TableGradArgs a{};
  a.rows = (int)rows;
  a.cols = cols;
  char* at = static_cast<char*>(scratch);
  auto add = [&](const int64_t* index, void* out, int n, float s) {
    Table& t = a.table[a.tables++];
    t.out = out;
    t.vocab = n;
    t.scale = s;
    t.seq = seq;
    t.batch = index ? 1 : (int)(rows / seq);
    t.partial = reinterpret_cast<float*>(at);
    at += partialBytes(rows, cols);
    if (index == nullptr) return 0;
    void* sorted = at;
    at += round16(8 * rows);
    int* skey = reinterpret_cast<int*>(at);
    at += round16(4 * rows);
    int* perm = reinterpret_cast<int*>(at);
    at += round16(4 * rows);
    t.skey = skey;
    t.perm = perm;
    return sortTokens(index, sorted, skey, perm, (int)rows, n, stream);
  };
  if (dw)
    if (int rc = add(token, dw, vocab, scale)) return rc;
  if (dp)
    if (int rc = add(position, dp, context, 1.0f)) return rc;
  auto f = g_f32 ? (d_f32 ? tableGradients<float, float> : tableGradients<float, uint16_t>)
                 : (d_f32 ? tableGradients<uint16_t, float> : tableGradients<uint16_t, uint16_t>);
  return f(g, a, stream);
}
