// Tokens sorted by expert and back, weights applied, and the gradients.
//
//   dispatch            sorted[position[t,k]] = x[t]
//   combine             out[t] = sum_k w[t,k] rows[position[t,k]]
//   dispatch gradient   dx[t] = sum_k g[position[t,k]]
//   combine gradient    drows[position[t,k]] = w[t,k] g[t],  dw[t,k] = <g[t], rows[position[t,k]]>
//
// Every slot, dropped ones too, has a sorted row of its own (ops_sort.cu puts the dropped
// ones last), so all of them go by the token: a token's row is read once and its slots'
// rows are written, or the other way round, with no atomics, no fill and no count on the
// host.  Bound by HBM: tokens x slots x dim elements one way, tokens x dim the other.
//
// The routing is the caller's: a position outside [0, tokens x slots), which purin_route does
// not make, is neither read nor written; its slot counts as dropped.
#include "ops_sort.cuh"

namespace purin {
namespace ops {
namespace {

constexpr int kThreads = 256;

// Work items are (token, C packs of V columns); item i of a token's n items has the packs i,
// i + n, ..., so that adjacent threads have adjacent packs.  Where a pack is one element,
// several of them keep enough reads in flight (4099 tokens x 3 slots x 1031 float32: spread 21 us
// against 28, gather 29 against 35, the gradient of combine 33 against 41).  Of 16384 tokens x 8
// slots x 2048 bf16 spread moves 5.9 TB/s, gather 5.3.
template <int V>
constexpr int kPacksAtOnce = V == 1 ? 4 : 1;

// Sorted rows in use, at most all of them.
__device__ __forceinline__ int32_t kept_of(const int32_t* kept_rows, int32_t rows) {
  return max(0, min(*kept_rows, rows));
}
__device__ __forceinline__ bool below(int32_t r, int32_t end) { return uint32_t(r) < uint32_t(end); }

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
spread_kernel(const int32_t* position, const int32_t* kept_rows, int64_t tokens, int slots,
              int64_t packs, const T* x, int64_t stride, T* out) {
  constexpr int C = kPacksAtOnce<V>;
  const int32_t rows = int32_t(tokens * slots), kept = kept_of(kept_rows, rows);
  const int64_t items = (packs + C - 1) / C, total = tokens * items;
  const bool fits32 = total <= INT32_MAX;
  for (int64_t at = int64_t(blockIdx.x) * kThreads + threadIdx.x; at < total;
       at += int64_t(gridDim.x) * kThreads) {
    int64_t t, c;
    divide(at, items, fits32, t, c);
    Pack<T, V> p[C], zero;
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (C == 1 || c + j * items < packs) p[j] = *reinterpret_cast<const Pack<T, V>*>(x + t * stride + (c + j * items) * V);
#pragma unroll
    for (int i = 0; i < V; ++i) zero.v[i] = narrow<T>(acc_t<T>(0));
#pragma unroll 4
    for (int k = 0; k < slots; ++k) {
      const int32_t r = position[t * slots + k];
      const bool inside = below(r, rows);
      Pack<T, V>* to = reinterpret_cast<Pack<T, V>*>(out) + int64_t(r) * packs + c;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const Pack<T, V> q = r < kept ? p[j] : zero;
        if (inside && (C == 1 || c + j * items < packs)) to[j * items] = q;
      }
    }
  }
}

template <typename T, int V, typename W, bool kWeighted>
__global__ void __launch_bounds__(kThreads, 4)
gather_kernel(const int32_t* position, const int32_t* kept_rows, int64_t tokens, int slots,
              int64_t packs, const T* rows, int64_t stride, const W* weights, T* out) {
  using A = acc_t<T>;
  constexpr int C = kPacksAtOnce<V>;
  const int32_t kept = kept_of(kept_rows, int32_t(tokens * slots));
  const int64_t items = (packs + C - 1) / C, total = tokens * items;
  const bool fits32 = total <= INT32_MAX;
  for (int64_t at = int64_t(blockIdx.x) * kThreads + threadIdx.x; at < total;
       at += int64_t(gridDim.x) * kThreads) {
    int64_t t, c;
    divide(at, items, fits32, t, c);
    A sum[C][V];
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[j][i] = A(0);
    constexpr int kAhead = 4;  // rows loaded at a time
    for (int first = 0; first < slots; first += kAhead) {
      int32_t r[kAhead];
      Pack<T, V> p[kAhead][C];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        r[k] = first + k < slots ? position[t * slots + first + k] : -1;
        // A dropped slot's row and weight may hold anything: they are not read.
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (below(r[k], kept) && (C == 1 || c + j * items < packs))
            p[k][j] = *reinterpret_cast<const Pack<T, V>*>(rows + r[k] * stride + (c + j * items) * V);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (!below(r[k], kept)) continue;
        const A w = kWeighted ? A(weights[t * slots + first + k]) : A(1);
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) sum[j][i] += w * A(widen(p[k][j].v[i]));
      }
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (C > 1 && c + j * items >= packs) continue;
      Pack<T, V> q;
#pragma unroll
      for (int i = 0; i < V; ++i) q.v[i] = narrow<T>(sum[j][i]);
      reinterpret_cast<Pack<T, V>*>(out)[t * packs + c + j * items] = q;
    }
  }
}

// G threads per token, a pack each at a time, so that a token's slots are all in flight; its
// dot products are sums over the G threads.
// Four slots at a time and four blocks per SM: eight slots cost registers, and fewer blocks
// (or more, with spills) hide less of the reads: 205 us against 245 to 610 for 16384 tokens
// of 8 slots and 2048 bf16 columns, 5.6 TB/s.
constexpr int kSlotsAtOnce = 4;

template <typename T, int V, typename W, int G>
__global__ void __launch_bounds__(kThreads, 4)
combine_backward_kernel(const int32_t* position, const int32_t* kept_rows, int64_t tokens,
                        int slots, int64_t packs, const T* grad, int64_t grad_stride,
                        const T* rows, int64_t stride, const W* weights, T* grad_rows,
                        W* grad_weights) {
  using A = acc_t<T>;
  constexpr int kTokens = kThreads / G, kWarps = G / 32, C = kPacksAtOnce<V>;
  __shared__ A part[kThreads / 32][kSlotsAtOnce];
  const int32_t all = int32_t(tokens * slots), kept = kept_of(kept_rows, all);
  const int lane = threadIdx.x & 31, in = threadIdx.x % G, warp = threadIdx.x >> 5;
  for (int64_t t0 = int64_t(blockIdx.x) * kTokens; t0 < tokens; t0 += int64_t(gridDim.x) * kTokens) {
    const int64_t t = t0 + threadIdx.x / G;
    const bool real_token = t < tokens;
    for (int first = 0; first < slots; first += kSlotsAtOnce) {
      int32_t r[kSlotsAtOnce];
      A dot[kSlotsAtOnce];
#pragma unroll
      for (int k = 0; k < kSlotsAtOnce; ++k) {
        r[k] = real_token && first + k < slots ? position[t * slots + first + k] : -1;
        if (r[k] >= all) r[k] = -1;
        dot[k] = A(0);
      }
      for (int64_t c = in; real_token && c < packs; c += G * C) {
        Pack<T, V> g[C];
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (c + j * G < packs) g[j] = *reinterpret_cast<const Pack<T, V>*>(grad + t * grad_stride + (c + j * G) * V);
        if (grad_weights) {
          Pack<T, V> p[kSlotsAtOnce][C];
#pragma unroll
          for (int k = 0; k < kSlotsAtOnce; ++k)
#pragma unroll
            for (int j = 0; j < C; ++j)
              if (r[k] >= 0 && r[k] < kept && c + j * G < packs)
                p[k][j] = *reinterpret_cast<const Pack<T, V>*>(rows + r[k] * stride + (c + j * G) * V);
#pragma unroll
          for (int k = 0; k < kSlotsAtOnce; ++k)
#pragma unroll
            for (int j = 0; j < C; ++j)
              if (r[k] >= 0 && r[k] < kept && c + j * G < packs) {
#pragma unroll
                for (int i = 0; i < V; ++i) dot[k] += A(widen(g[j].v[i])) * A(widen(p[k][j].v[i]));
              }
        }
        if (grad_rows) {
#pragma unroll
          for (int k = 0; k < kSlotsAtOnce; ++k) {
            if (r[k] < 0) continue;
            const bool real = r[k] < kept;
            const A w = real ? A(weights[t * slots + first + k]) : A(0);
#pragma unroll
            for (int j = 0; j < C; ++j) {
              if (c + j * G >= packs) continue;
              Pack<T, V> q;
#pragma unroll
              for (int i = 0; i < V; ++i) q.v[i] = narrow<T>(real ? w * A(widen(g[j].v[i])) : A(0));
              reinterpret_cast<Pack<T, V>*>(grad_rows)[r[k] * packs + c + j * G] = q;
            }
          }
        }
      }
      if (grad_weights) {
#pragma unroll
        for (int k = 0; k < kSlotsAtOnce; ++k) {
#pragma unroll
          for (int d = 16; d; d >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], d);
          if constexpr (kWarps == 1) {
            if (lane == 0 && real_token && first + k < slots) grad_weights[t * slots + first + k] = W(dot[k]);
          } else {
            if (lane == 0) part[warp][k] = dot[k];
          }
        }
        if constexpr (kWarps > 1) {
          __syncthreads();
          if (in < kSlotsAtOnce && real_token && first + in < slots) {
            A sum = A(0);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += part[warp + w][in];  // in < 4: the token's first warp
            grad_weights[t * slots + first + in] = W(sum);
          }
          __syncthreads();
        }
      }
    }
  }
}

int32_t check_route(const PurinRouteArgs* a) {
  if (!a) return invalid("route: null arguments");
  if (a->tokens < 0 || a->slots < 1 || a->num_experts < 1) return invalid("route: invalid sizes");
  if (a->num_experts >= INT32_MAX || a->tokens > INT32_MAX / a->slots)
    return set_error(PURIN_ERR_UNSUPPORTED, "route: tokens x slots must be below 2^31");
  return PURIN_OK;
}

int32_t check_rows(const PurinRouteRowsArgs* a, bool token_rows, bool sorted_rows) {
  if (!a) return invalid("route rows: null arguments");
  if (!known_dtype(a->dtype)) return invalid("route rows: unknown element type");
  if (a->tokens < 0 || a->slots < 1 || a->num_experts < 1 || a->dim < 1)
    return invalid("route rows: invalid sizes");
  if (a->slots > INT32_MAX || a->tokens > INT32_MAX / a->slots)
    return set_error(PURIN_ERR_UNSUPPORTED, "route rows: tokens x slots must be below 2^31");
  if (!a->offsets || (a->tokens && !a->position)) return invalid("route rows: null routing");
  if (a->tokens && token_rows && !a->token_rows) return invalid("route rows: null token rows");
  if (a->tokens && sorted_rows && !a->sorted_rows) return invalid("route rows: null sorted rows");
  if (a->token_stride < 0 || a->sorted_stride < 0) return invalid("route rows: negative stride");
  return PURIN_OK;
}

template <typename F>
int32_t with_weights(int32_t dtype, F&& f) {
  if (dtype == PURIN_OPS_FLOAT64) return f(double());
  if (dtype == PURIN_OPS_FLOAT32) return f(float());
  return invalid("route rows: weights must be float32 or float64");
}

}  // namespace
}  // namespace ops
}  // namespace purin

using namespace purin::ops;
using purin::set_error;

extern "C" int32_t purin_route_workspace_size(const PurinRouteArgs* a, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_route(a)) return bad;
    if (!bytes) return invalid("route: null arguments");
    *bytes = key_sort_workspace(a->tokens * a->slots, a->num_experts);
    return PURIN_OK;
  });
}

extern "C" int32_t purin_route(const PurinRouteArgs* a, void* workspace, size_t workspace_bytes,
                               void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_route(a)) return bad;
    const int64_t n = a->tokens * a->slots;
    if (!a->offsets || (n && (!a->experts || !a->position || !a->source)))
      return invalid("route: null experts, offsets, position or source");
    const size_t need = key_sort_workspace(n, a->num_experts);
    if (need && (!workspace || workspace_bytes < need))
      return set_error(PURIN_ERR_WORKSPACE, "route: workspace too small");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    KeySort sort;
    sort.ids = a->experts;
    sort.ids_64bit = a->experts_64bit != 0;
    sort.n = n;
    sort.range = a->num_experts;
    sort.source = a->source;
    sort.position = a->position;
    sort.offsets = a->offsets;
    return cuda_status(key_sort(sort, workspace, static_cast<cudaStream_t>(stream)));
  });
}

extern "C" int32_t purin_route_spread(const PurinRouteRowsArgs* a, void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_rows(a, true, false)) return bad;
    if (a->tokens == 0) return PURIN_OK;
    if (!a->sorted_out) return invalid("route rows: null output");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    return with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      auto s = static_cast<cudaStream_t>(stream);
      auto x = static_cast<const T*>(a->token_rows);
      auto out = static_cast<T*>(a->sorted_out);
      const int32_t* kept = a->offsets + a->num_experts;
      const bool wide = packable(x, a->token_stride, a->dim, sizeof(T), V) &&
                        packable(out, a->dim, a->dim, sizeof(T), V);
      const int64_t packs = wide ? a->dim / V : a->dim;
      const unsigned grid = grid_for(a->tokens * (wide ? packs : ceil_div(packs, 4)), kThreads, sm_count(a->device));
      if (wide)
        spread_kernel<T, V><<<grid, kThreads, 0, s>>>(a->position, kept, a->tokens, int(a->slots), packs, x, a->token_stride, out);
      else
        spread_kernel<T, 1><<<grid, kThreads, 0, s>>>(a->position, kept, a->tokens, int(a->slots), packs, x, a->token_stride, out);
      return launched();
    });
  });
}

extern "C" int32_t purin_route_gather(const PurinRouteRowsArgs* a, void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_rows(a, false, true)) return bad;
    if (a->tokens == 0) return PURIN_OK;
    if (!a->token_out) return invalid("route rows: null output");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    return with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      auto s = static_cast<cudaStream_t>(stream);
      auto rows = static_cast<const T*>(a->sorted_rows);
      auto out = static_cast<T*>(a->token_out);
      const int32_t* kept = a->offsets + a->num_experts;
      const bool wide = packable(rows, a->sorted_stride, a->dim, sizeof(T), V) &&
                        packable(out, a->dim, a->dim, sizeof(T), V);
      const int64_t packs = wide ? a->dim / V : a->dim;
      const unsigned grid = grid_for(a->tokens * (wide ? packs : ceil_div(packs, 4)), kThreads, sm_count(a->device));
      auto launch = [&](auto w, auto weighted) {
        using W = decltype(w);
        auto weights = static_cast<const W*>(a->weights);
        if (wide)
          gather_kernel<T, V, W, decltype(weighted)::value><<<grid, kThreads, 0, s>>>(
              a->position, kept, a->tokens, int(a->slots), packs, rows, a->sorted_stride, weights, out);
        else
          gather_kernel<T, 1, W, decltype(weighted)::value><<<grid, kThreads, 0, s>>>(
              a->position, kept, a->tokens, int(a->slots), packs, rows, a->sorted_stride, weights, out);
        return launched();
      };
      if (!a->weights) return launch(float(), std::false_type());
      return with_weights(a->weights_dtype, [&](auto w) { return launch(w, std::true_type()); });
    });
  });
}

extern "C" int32_t purin_route_combine_backward(const PurinRouteRowsArgs* a, void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_rows(a, true, a && a->grad_weights)) return bad;
    if (a->tokens == 0) return PURIN_OK;
    if (!a->weights) return invalid("route rows: null weights");
    if (!a->sorted_out && !a->grad_weights) return invalid("route rows: null output");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    return with_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      auto s = static_cast<cudaStream_t>(stream);
      auto grad = static_cast<const T*>(a->token_rows);
      auto rows = static_cast<const T*>(a->sorted_rows);
      auto grad_rows = static_cast<T*>(a->sorted_out);
      const int32_t* kept = a->offsets + a->num_experts;
      const bool wide = packable(grad, a->token_stride, a->dim, sizeof(T), V) &&
                        packable(grad_rows, a->dim, a->dim, sizeof(T), V) &&
                        (!a->grad_weights || packable(rows, a->sorted_stride, a->dim, sizeof(T), V));
      const int64_t packs = wide ? a->dim / V : a->dim;
      return with_weights(a->weights_dtype, [&](auto w) {
        using W = decltype(w);
        auto weights = static_cast<const W*>(a->weights);
        auto grad_weights = static_cast<W*>(a->grad_weights);
        auto launch = [&](auto kernel, int group) {
          const unsigned grid = grid_for(a->tokens, kThreads / group, sm_count(a->device));
          kernel<<<grid, kThreads, 0, s>>>(a->position, kept, a->tokens, int(a->slots), packs, grad,
                                           a->token_stride, rows, a->sorted_stride, weights, grad_rows,
                                           grad_weights);
          return launched();
        };
        if (wide)
          return packs > 32 ? launch(combine_backward_kernel<T, V, W, 256>, 256)
                            : launch(combine_backward_kernel<T, V, W, 32>, 32);
        return packs > 32 ? launch(combine_backward_kernel<T, 1, W, 256>, 256)
                          : launch(combine_backward_kernel<T, 1, W, 32>, 32);
      });
    });
  });
}
