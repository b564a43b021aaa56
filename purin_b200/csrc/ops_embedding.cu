// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[i] = scale * table[ids[i]]             (zero row for an id without a row)
//   grad_table[v] = scale * sum_{i: ids[i] = v} grad_out[i], in the order of i
//
// Both are bound by HBM: the lookup moves each row once, the gradient reads every row of
// grad_out once and writes every row of the table once.
#include <algorithm>

#include "ops_sort.cuh"

namespace purin {
namespace ops {
namespace {

constexpr int kThreads = 256;

struct Ids {
  const void* ids;
  bool is_64bit;
  int64_t vocab, padding;
  __device__ __forceinline__ int64_t row(int64_t i) const {  // -1: no row
    const int64_t id = is_64bit ? static_cast<const int64_t*>(ids)[i]
                                : int64_t(static_cast<const int32_t*>(ids)[i]);
    return id >= 0 && id < vocab && id != padding ? id : -1;
  }
};

// Rows of more than 32 packs, one warp per token: the id is read once and a row's packs are in
// flight together (4099 x 771 float32: 6.6 us, one pack a thread 12.6; 32768 x 2048 bf16 with
// streaming stores 34.5 us, 5.7 TB/s, without 42).
template <typename T, int V, bool kStream>
__global__ void __launch_bounds__(kThreads)
lookup_kernel(Ids ids, const T* table, int64_t stride, int64_t tokens, int64_t packs,
              acc_t<T> scale, T* out) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * (kThreads / 32);
  for (int64_t i = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); i < tokens; i += warps) {
    const int64_t row = ids.row(i);
    const Pack<T, V>* from = reinterpret_cast<const Pack<T, V>*>(table + (row >= 0 ? row * stride : 0));
    Pack<T, V>* to = reinterpret_cast<Pack<T, V>*>(out) + i * packs;
    for (int64_t c = lane; c < packs; c += 32 * kAhead) {
      Pack<T, V> p[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (row >= 0 && c + 32 * j < packs) p[j] = from[c + 32 * j];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (c + 32 * j >= packs) break;
#pragma unroll
        for (int k = 0; k < V; ++k)
          p[j].v[k] = narrow<T>(row >= 0 ? scale * widen(p[j].v[k]) : acc_t<T>(0));
        store_pack<kStream>(to + c + 32 * j, p[j]);
      }
    }
  }
}

// Shorter rows, one pack a thread: adjacent threads write adjacent packs whatever the row's
// length (100000 x 9 float32: 6.3 us, a part of a warp per token 11.7).
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
lookup_short_kernel(Ids ids, const T* table, int64_t stride, int64_t tokens, int64_t packs,
                    acc_t<T> scale, T* out) {
  const int64_t total = tokens * packs;
  const bool fits32 = total <= INT32_MAX;
  for (int64_t at = int64_t(blockIdx.x) * kThreads + threadIdx.x; at < total;
       at += int64_t(gridDim.x) * kThreads) {
    int64_t i, c;
    divide(at, packs, fits32, i, c);
    const int64_t row = ids.row(i);
    Pack<T, V> p;
    if (row >= 0) p = *reinterpret_cast<const Pack<T, V>*>(table + row * stride + c * V);
#pragma unroll
    for (int k = 0; k < V; ++k) p.v[k] = narrow<T>(row >= 0 ? scale * widen(p.v[k]) : acc_t<T>(0));
    reinterpret_cast<Pack<T, V>*>(out)[at] = p;
  }
}

// ---- gradient ------------------------------------------------------------------------
// The sorted tokens are cut into chunks of kChunk places, whatever their ids: a frequent
// token's sum is spread over many blocks, a block of rare tokens writes many rows.  A run
// of one id that lies within a chunk is summed and written; a run that crosses a chunk's
// edge leaves a partial sum per chunk, and join_kernel adds a run's partial sums in order.
// Rows without a token are written as zeros by further blocks of the same launch, which
// find their rows' tokens by a search in the sorted ids.
constexpr int kChunk = 64;
constexpr int kMostRows = 1024;  // table rows of a block that writes zeros

// First place whose key is not below `value`; all lanes of a warp take part (a 33-ary search).
__device__ __forceinline__ int64_t lower_bound(const int32_t* key, int64_t n, int32_t value) {
  const int lane = threadIdx.x & 31;
  int64_t low = 0, high = n;  // keys before low are below value, keys from high on are not
  while (low < high) {
    const int64_t width = high - low;
    const int64_t at = low + width * (lane + 1) / 33;  // ascending over the lanes, below high
    const unsigned below = __ballot_sync(0xffffffffu, key[at] < value);
    const int count = __popc(below);  // the first `count` lanes are below
    const int64_t left = __shfl_sync(0xffffffffu, at, count ? count - 1 : 0);
    const int64_t right = __shfl_sync(0xffffffffu, at, count < 32 ? count : 31);
    if (count) low = left + 1;
    if (count < 32) high = right;
  }
  return low;
}

template <typename T, int V, int VT, bool kStream>
__global__ void __launch_bounds__(kThreads, 4)
gradient_kernel(const int32_t* key, const int32_t* source, int64_t tokens, int32_t vocab,
                const T* grad, int64_t stride, int64_t dim, acc_t<T> scale, T* table,
                acc_t<T>* partial, int64_t chunk_blocks, int column_blocks, int rows_per_block) {
  using A = acc_t<T>;
  wait_for_previous();
  let_next_start();
  if (int64_t(blockIdx.x) >= chunk_blocks) {
    __shared__ uint8_t present[kMostRows];
    __shared__ int64_t bound[2];
    const int64_t first = (blockIdx.x - chunk_blocks) * rows_per_block;
    const int rows = int(min(int64_t(rows_per_block), vocab - first));
    for (int r = threadIdx.x; r < rows; r += kThreads) present[r] = 0;
    if (threadIdx.x < 64) {
      const int which = threadIdx.x >> 5;
      const int64_t at = lower_bound(key, tokens, int32_t(first + (which ? rows : 0)));
      if ((threadIdx.x & 31) == 0) bound[which] = at;
    }
    __syncthreads();
    for (int64_t i = bound[0] + threadIdx.x; i < bound[1]; i += kThreads) present[key[i] - first] = 1;
    __syncthreads();
    Pack<T, VT> zero;
#pragma unroll
    for (int k = 0; k < VT; ++k) zero.v[k] = narrow<T>(A(0));
    const int64_t packs = dim / VT;
    // Threads go along a row, or over several short ones.
    const int across = packs < kThreads ? int(packs) : kThreads;
    const int down = kThreads / across;
    const int r0 = threadIdx.x / across, c0 = threadIdx.x % across;
    if (r0 >= down) return;
    for (int r = r0; r < rows; r += down) {
      if (present[r]) continue;
      Pack<T, VT>* to = reinterpret_cast<Pack<T, VT>*>(table + (first + r) * dim);
      for (int64_t c = c0; c < packs; c += across) store_pack<kStream>(to + c, zero);
    }
    return;
  }
  const int64_t chunk = blockIdx.x / column_blocks;
  const int64_t column = (int64_t(blockIdx.x % column_blocks) * kThreads + threadIdx.x) * V;
  if (column >= dim) return;
  const int64_t begin = chunk * kChunk;
  const int64_t end = min(begin + kChunk, tokens);
  A sum[V];
#pragma unroll
  for (int k = 0; k < V; ++k) sum[k] = A(0);
  bool head = begin > 0 && key[begin] == key[begin - 1];  // this run started in an earlier chunk
  constexpr int kAhead = 4;  // rows loaded at a time
  for (int64_t i0 = begin; i0 < end; i0 += kAhead) {
    Pack<T, V> row[kAhead];
    int32_t id[kAhead + 1];
#pragma unroll
    for (int j = 0; j <= kAhead; ++j) id[j] = i0 + j < end ? key[i0 + j] : -1;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j < end && id[j] < vocab)
        row[j] = *reinterpret_cast<const Pack<T, V>*>(grad + source[i0 + j] * stride + column);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j >= end || id[j] >= vocab) break;  // ids without a row sort last
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += widen(row[j].v[k]);
      if (id[j + 1] == id[j]) continue;
      const bool goes_on = i0 + j + 1 == end && end < tokens && key[end] == id[j];
      if (head || goes_on) {
        A* to = partial + (chunk * 2 + (head ? 0 : 1)) * dim + column;
#pragma unroll
        for (int k = 0; k < V; ++k) to[k] = sum[k];
      } else {
        Pack<T, V> q;
#pragma unroll
        for (int k = 0; k < V; ++k) q.v[k] = narrow<T>(scale * sum[k]);
        store_pack<kStream>(reinterpret_cast<Pack<T, V>*>(table + int64_t(id[j]) * dim + column), q);
      }
      head = false;
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = A(0);
    }
  }
}

// Blocks per chunk whose last run starts in it and goes on: they add the run's partial sums.
template <typename T>
__global__ void __launch_bounds__(kThreads)
join_kernel(const int32_t* key, int64_t tokens, int32_t vocab, int64_t dim, acc_t<T> scale,
            T* table, const acc_t<T>* partial, int column_blocks) {
  using A = acc_t<T>;
  wait_for_previous();
  const int64_t chunk = blockIdx.x / column_blocks, begin = chunk * kChunk, end = begin + kChunk;
  if (end >= tokens) return;
  const int32_t id = key[end - 1];
  if (id >= vocab || key[end] != id) return;
  if (begin > 0 && key[begin - 1] == id) return;  // started earlier
  // Last chunk that holds part of the run.
  const int64_t last = (end + lower_bound(key + end, tokens - end, id + 1) - 1) / kChunk;
  const int64_t c = int64_t(blockIdx.x % column_blocks) * kThreads + threadIdx.x;
  if (c >= dim) return;
  A sum = partial[(chunk * 2 + 1) * dim + c];
#pragma unroll 8
  for (int64_t k = chunk + 1; k <= last; ++k) sum += partial[k * 2 * dim + c];
  table[int64_t(id) * dim + c] = narrow<T>(scale * sum);
}

int32_t check(const PurinEmbeddingArgs* a, bool backward) {
  if (!a) return invalid("embedding: null arguments");
  if (!known_dtype(a->dtype)) return invalid("embedding: unknown element type");
  if (a->tokens < 0 || a->vocab < 1 || a->dim < 1) return invalid("embedding: invalid sizes");
  if (a->tokens > INT32_MAX || a->vocab >= INT32_MAX || a->dim > INT32_MAX)
    return set_error(PURIN_ERR_UNSUPPORTED, "embedding: sizes must be below 2^31");
  if (a->tokens && !a->ids) return invalid("embedding: null ids");
  if (!backward && a->tokens && (!a->table || !a->out)) return invalid("embedding: null table or out");
  if (!backward && a->table_stride < 0) return invalid("embedding: negative table stride");
  if (backward && (!a->grad_table || (a->tokens && !a->grad_out)))
    return invalid("embedding: null grad_table or grad_out");
  if (backward && a->tokens && a->grad_out_stride < 0)
    return invalid("embedding: negative grad_out stride");
  return PURIN_OK;
}

struct BackwardLayout {
  size_t source, key, partial, sort, total;
  int64_t chunks;
};
BackwardLayout backward_layout(const PurinEmbeddingArgs* a) {
  BackwardLayout l;
  const size_t n = size_t(a->tokens);
  l.chunks = ceil_div(a->tokens, kChunk);
  l.source = 0;
  l.key = l.source + align256(n * 4);
  l.partial = l.key + align256(n * 4);
  l.sort = l.partial + align256(size_t(l.chunks) * 2 * a->dim * (a->dtype == PURIN_OPS_FLOAT64 ? 8 : 4));
  l.total = l.sort + key_sort_workspace(a->tokens, a->vocab);
  return l;
}

}  // namespace
}  // namespace ops
}  // namespace purin

using namespace purin::ops;
using purin::set_error;

extern "C" int32_t purin_embedding_forward(const PurinEmbeddingArgs* a, void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check(a, false)) return bad;
    if (a->tokens == 0) return PURIN_OK;
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    const Ids ids{a->ids, a->ids_64bit != 0, a->vocab, a->padding};
    return with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      constexpr int W = 16 / sizeof(T);
      const bool wide = packable(a->table, a->table_stride, a->dim, sizeof(T), W) &&
                        packable(a->out, a->dim, a->dim, sizeof(T), W);
      const int64_t packs = wide ? a->dim / W : a->dim;
      auto s = static_cast<cudaStream_t>(stream);
      auto table = static_cast<const T*>(a->table);
      auto out = static_cast<T*>(a->out);
      const acc_t<T> scale = acc_t<T>(a->scale);
      const int sms = sm_count(a->device);
      const bool stream_out = a->tokens * a->dim * int64_t(sizeof(T)) > kStreamBytes;
      auto launch = [&](auto kernel, int64_t items, int64_t per_block) {
        kernel<<<grid_for(items, per_block, sms), kThreads, 0, s>>>(ids, table, a->table_stride, a->tokens, packs,
                                                                   scale, out);
      };
      if (packs <= 32)
        launch(wide ? lookup_short_kernel<T, W> : lookup_short_kernel<T, 1>, a->tokens * packs, kThreads);
      else if (wide)
        launch(stream_out ? lookup_kernel<T, W, true> : lookup_kernel<T, W, false>, a->tokens, kThreads / 32);
      else
        launch(lookup_kernel<T, 1, false>, a->tokens, kThreads / 32);
      return launched();
    });
  });
}

extern "C" int32_t purin_embedding_backward_workspace_size(const PurinEmbeddingArgs* a, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (!a || !bytes) return invalid("embedding: null arguments");
    if (!known_dtype(a->dtype)) return invalid("embedding: unknown element type");
    if (a->tokens < 0 || a->vocab < 1 || a->dim < 1) return invalid("embedding: invalid sizes");
    *bytes = backward_layout(a).total;
    return PURIN_OK;
  });
}

extern "C" int32_t purin_embedding_backward(const PurinEmbeddingArgs* a, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check(a, true)) return bad;
    const BackwardLayout l = backward_layout(a);
    if (l.total && (!workspace || workspace_bytes < l.total))
      return set_error(PURIN_ERR_WORKSPACE, "embedding: workspace too small");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    auto s = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    auto source = reinterpret_cast<int32_t*>(ws + l.source);
    auto key = reinterpret_cast<int32_t*>(ws + l.key);
    if (a->tokens) {
      KeySort sort;
      sort.ids = a->ids;
      sort.ids_64bit = a->ids_64bit != 0;
      sort.n = a->tokens;
      sort.range = a->vocab;
      sort.skip = a->padding;
      sort.source = source;
      sort.key = key;
      if (cudaError_t e = key_sort(sort, ws + l.sort, s)) return cuda_status(e);
    }
    return with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      using A = acc_t<T>;
      constexpr int W = 16 / sizeof(T);
      auto grad = static_cast<const T*>(a->grad_out);
      auto table = static_cast<T*>(a->grad_table);
      auto partial = reinterpret_cast<A*>(ws + l.partial);
      const bool wide_table = packable(table, a->dim, a->dim, sizeof(T), W);
      const bool wide = wide_table && packable(grad, a->grad_out_stride, a->dim, sizeof(T), W);
      const A scale = A(a->scale);
      const int64_t columns = ceil_div(a->dim, int64_t(kThreads) * (wide ? W : 1));
      const int64_t chunk_blocks = l.chunks * columns;
      // Rows per block that writes zeros: at least 64 KB, and no more blocks than run at once, so
      // that the search (some 2 us) is made once per block's share.
      int64_t rows = ceil_div(65536, a->dim * int64_t(sizeof(T)));
      rows = std::max(rows, ceil_div(a->vocab, int64_t(sm_count(a->device)) * 4));
      rows = std::min<int64_t>(rows, kMostRows);
      const int64_t blocks = chunk_blocks + ceil_div(a->vocab, rows);
      const int64_t join_columns = ceil_div(a->dim, kThreads);
      if (blocks > INT32_MAX || l.chunks * join_columns > INT32_MAX)
        return set_error(PURIN_ERR_UNSUPPORTED, "embedding: too large");
      auto launch = [&](auto kernel) {
        return launch_after(kernel, dim3(unsigned(blocks)), dim3(kThreads), 0, s, key, source, a->tokens,
                            int32_t(a->vocab), grad, a->grad_out_stride, a->dim, scale, table, partial,
                            chunk_blocks, int(columns), int(rows));
      };
      const bool stream_out = a->vocab * a->dim * int64_t(sizeof(T)) > kStreamBytes;  // 160 us against 169
      const cudaError_t e =
          wide ? launch(stream_out ? gradient_kernel<T, W, W, true> : gradient_kernel<T, W, W, false>)
          : wide_table ? launch(stream_out ? gradient_kernel<T, 1, W, true> : gradient_kernel<T, 1, W, false>)
                       : launch(gradient_kernel<T, 1, 1, false>);
      if (e != cudaSuccess) return cuda_status(e);
      if (l.chunks > 1)
        return cuda_status(launch_after(join_kernel<T>, dim3(unsigned(l.chunks * join_columns)), dim3(kThreads), 0,
                                        s, key, a->tokens, int32_t(a->vocab), a->dim, scale, table, partial,
                                        int(join_columns)));
      return launched();
    });
  });
}
