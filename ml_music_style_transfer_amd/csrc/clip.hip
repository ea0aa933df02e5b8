// Global gradient norm over many tensors, clipping, and Adam with the clip inside the update.
//
//   n = sqrt(sum_i g_i^2) over every element of every tensor;  c = min(1, max_norm / (n + 1e-6))
//   scale: g <- c g (in place);  adam: the update of adam_kernel (norm.hip) on c g, g left as it is
//
// A launch takes the addresses by value (a table in the kernel arguments: nothing to upload, and a
// captured graph keeps them). Each tensor is cut into chunks; workgroup k takes the launch's chunks
// k, k + gridDim.x, ... All of it is bound by HBM. Small chunks in order keep what is in flight close
// together in memory: over 726 M parameters, chunks of 16384 / 4096 / 1024 elements run the norm in
// 472 / 459 / 555 us (a lookup a chunk; 6.3 TB/s) and Adam in 3.81 / 3.50 / 3.37 ms (ten calls in a row, 6.0
// TB/s; its predecessor without the clip 4.11 ms on the same card; without nontemporal access 3.96 -> 3.77
// at most). Traced between other kernels Adam's median is 3.43 to 3.58 ms, 5.7 to 5.9 TB/s.
#include <new>

#include "common.h"

namespace {

constexpr int kChunk = 4096;       // elements: 4 float4 steps of a 256-thread workgroup
constexpr int kAdamChunk = 1024;   // one float4 of each tensor a thread
constexpr int kNormBlocks = 2048;  // workgroups, and partial sums, of a launch of the norm
constexpr int kTensors = 160;      // table entries: 160 x 21 bytes of kernel arguments (limit 4 KB)
constexpr int kAdamTensors = 80;   // 80 x 44 bytes

struct Table {
  void* p[kTensors];
  long long n[kTensors];
  int first[kTensors];  // index of the tensor's first chunk in this launch
  unsigned char type[kTensors];
  int count, chunks;
};

struct AdamTable {
  float* p[kAdamTensors];
  const float* g[kAdamTensors];
  float* m[kAdamTensors];
  float* v[kAdamTensors];
  long long n[kAdamTensors];
  int first[kAdamTensors];
  int count, chunks;
};

// 16 bytes at the element's own alignment (gradients may be slices that start anywhere)
typedef float f32v __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16v __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16v __attribute__((ext_vector_type(8), aligned(2)));
template <typename T> struct VecOf;
template <> struct VecOf<float> { typedef f32v t; };
template <> struct VecOf<__bf16> { typedef bf16v t; };
template <> struct VecOf<_Float16> { typedef f16v t; };

// last entry of a launch's table whose first chunk is <= chunk
template <typename TB>
__device__ __forceinline__ int find(const TB& tb, int chunk) {
  int lo = 0, hi = tb.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tb.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Squares are summed in double: a float's square neither overflows nor underflows there, and a
// sum of 1e9 terms keeps more digits than the float that is returned.
template <typename T>
__device__ __forceinline__ double chunk_square(const T* g, int n) {
  typedef typename VecOf<T>::t V;
  constexpr int E = 16 / sizeof(T);
  double s = 0.0;
  const int nv = n / E;
  for (int i = threadIdx.x; i < nv; i += 256) {
    const V v = *reinterpret_cast<const V*>(g + (long long)i * E);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const double d = (double)(float)v[k];
      s = fma(d, d, s);
    }
  }
  const int i = nv * E + threadIdx.x;
  if (i < n) {
    const double d = (double)(float)g[i];
    s = fma(d, d, s);
  }
  return s;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, int n, float c) {
  typedef typename VecOf<T>::t V;
  constexpr int E = 16 / sizeof(T);
  const int nv = n / E;
  for (int i = threadIdx.x; i < nv; i += 256) {
    V v = *reinterpret_cast<const V*>(g + (long long)i * E);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = (T)((float)v[k] * c);  // the product in float, rounded once
    *reinterpret_cast<V*>(g + (long long)i * E) = v;
  }
  const int i = nv * E + threadIdx.x;
  if (i < n) g[i] = (T)((float)g[i] * c);
}

// sum over the workgroup's 256 threads, on thread 0
__device__ __forceinline__ double block_sum(double s) {
  __shared__ double red[4];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// torch's clip: a norm that is not a number gives a factor that is none either
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  const float c = max_norm / (norm + 1e-6f);
  return c >= 1.f ? 1.f : c;
}

__global__ __launch_bounds__(256) void norm_partial_kernel(const Table tb, double* __restrict__ part) {
  double s = 0.0;
  for (int c = blockIdx.x; c < tb.chunks; c += gridDim.x) {
    const int i = find(tb, c);
    const long long at = (long long)(c - tb.first[i]) * kChunk;
    const int n = (int)min((long long)kChunk, tb.n[i] - at);
    const int type = tb.type[i];
    if (type == MST_F32) s += chunk_square((const float*)tb.p[i] + at, n);
    else if (type == MST_BF16) s += chunk_square((const __bf16*)tb.p[i] + at, n);
    else s += chunk_square((const _Float16*)tb.p[i] + at, n);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void norm_final_kernel(const double* __restrict__ part, int np,
                                                         float* __restrict__ norm) {
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < np; i += 256) s += part[i];
  s = block_sum(s);
  if (threadIdx.x == 0) norm[0] = (float)sqrt(s);
}

// From the end to the start: what the norm read last is still in the 256 MB cache (90 M float32
// gradients, norm and scale: 208 -> 167 us; 726 M: 1533 -> 1508 us).
__global__ __launch_bounds__(256) void clip_scale_kernel(const Table tb, const float* __restrict__ norm,
                                                         float max_norm) {
  const float f = clip_factor(norm[0], max_norm);
  if (f == 1.f) return;  // under the limit: a product by one would give every value back
  for (int k = blockIdx.x; k < tb.chunks; k += gridDim.x) {
    const int c = tb.chunks - 1 - k, i = find(tb, c);
    const long long at = (long long)(c - tb.first[i]) * kChunk;
    const int n = (int)min((long long)kChunk, tb.n[i] - at);
    const int type = tb.type[i];
    if (type == MST_F32) chunk_scale((float*)tb.p[i] + at, n, f);
    else if (type == MST_BF16) chunk_scale((__bf16*)tb.p[i] + at, n, f);
    else chunk_scale((_Float16*)tb.p[i] + at, n, f);
  }
}

struct AdamK {
  float lr_step, b2, w1, w2, eps, bc2_sqrt;
};
// The sums are fused by hand: every element rounds alike, wherever it lies in a vector.
__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, const AdamK& k) {
#pragma clang fp contract(off)
  m = fmaf(k.w1, g - m, m);
  v = fmaf(k.w2, g * g, v * k.b2);
  p = fmaf(-k.lr_step, m / (sqrtf(v) / k.bc2_sqrt + k.eps), p);
}

__global__ __launch_bounds__(256) void adam_clip_kernel(const AdamTable tb, const float* __restrict__ norm,
                                                        float max_norm, AdamK k,
                                                        const float* __restrict__ hyper) {
  const float f = clip_factor(norm[0], max_norm);
  if (hyper) {
    k.lr_step = hyper[0];
    k.bc2_sqrt = hyper[1];
  }
  // one chunk a workgroup (the grid is tb.chunks)
  const int c = blockIdx.x, i = find(tb, c);
  const long long at = (long long)(c - tb.first[i]) * kAdamChunk;
  const int n = (int)min((long long)kAdamChunk, tb.n[i] - at), j = threadIdx.x * 4;
  float *p = tb.p[i] + at + j, *m = tb.m[i] + at + j, *v = tb.v[i] + at + j;
  const float* g = tb.g[i] + at + j;
  if (j + 4 <= n) {  // streamed once: nontemporal
    f32v pv = __builtin_nontemporal_load((f32v*)p), mv = __builtin_nontemporal_load((f32v*)m);
    f32v vv = __builtin_nontemporal_load((f32v*)v);
    const f32v gv = __builtin_nontemporal_load((const f32v*)g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float pe = pv[e], me = mv[e], ve = vv[e];
      adam_one(pe, gv[e] * f, me, ve, k);
      pv[e] = pe, mv[e] = me, vv[e] = ve;
    }
    __builtin_nontemporal_store(pv, (f32v*)p);
    __builtin_nontemporal_store(mv, (f32v*)m);
    __builtin_nontemporal_store(vv, (f32v*)v);
  } else {
    for (int e = 0; j + e < n; ++e) adam_one(p[e], g[e] * f, m[e], v[e], k);
  }
}

int size_of(int type) { return type == MST_F32 ? 4 : 2; }

// Chunks of a tensor, and workgroups of a launch: a grid has fewer than 2^32 threads. The chunks of
// kTensors such tensors, four times as long, are still an int.
constexpr int kMaxChunks = 0xffffff;

bool good_tensor(const void* p, int64_t n, int type) {
  if (n < 0 || n > (int64_t)kAdamChunk * kMaxChunks || type < MST_F32 || type > MST_F16) return false;
  return n == 0 || (p && (uintptr_t)p % size_of(type) == 0);
}

// Fills `tb` with entries from tensor *i on, until it has `cap` or the next would pass `most` chunks.
template <typename TB, typename F>
void fill(TB& tb, int cap, int chunk, int most, const int64_t* numel, int32_t count, int* i, F put) {
  tb.count = tb.chunks = 0;
  for (; *i < count && tb.count < cap; ++*i) {
    const int64_t c = (numel[*i] + chunk - 1) / chunk;
    if (c == 0) continue;
    if (c + tb.chunks > most) break;
    put(tb.count, *i);
    tb.n[tb.count] = numel[*i];
    tb.first[tb.count++] = tb.chunks;
    tb.chunks += (int)c;
  }
}

// Whether two of the ranges that a launch writes share memory: a value would be scaled (or stepped)
// by two workgroups at once. Heap sort by address, in place.
struct Range {
  uintptr_t a, b;
};
void sift(Range* r, int64_t i, int64_t n) {
  for (;;) {
    int64_t c = 2 * i + 1;
    if (c >= n) return;
    if (c + 1 < n && r[c].a < r[c + 1].a) ++c;
    if (r[i].a >= r[c].a) return;
    const Range t = r[i];
    r[i] = r[c], r[c] = t, i = c;
  }
}
bool overlap(Range* r, int64_t n) {
  for (int64_t i = n / 2 - 1; i >= 0; --i) sift(r, i, n);
  for (int64_t k = n - 1; k > 0; --k) {
    const Range t = r[0];
    r[0] = r[k], r[k] = t;
    sift(r, 0, k);
  }
  for (int64_t i = 1; i < n; ++i)
    if (r[i].a < r[i - 1].b) return true;
  return false;
}

}  // namespace

extern "C" {

size_t mst_grad_norm_workspace_size(int32_t count) {
  return count < 0 ? 0 : ((size_t)count / kTensors + 1) * kNormBlocks * sizeof(double);
}

int mst_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* types, int32_t count,
                  float* norm, void* workspace, size_t ws_bytes, void* stream) {
  MST_REQUIRE(count >= 0 && norm && (count == 0 || (grads && numel && types)));
  MST_REQUIRE(workspace && ws_bytes >= mst_grad_norm_workspace_size(count));
  for (int i = 0; i < count; ++i) MST_REQUIRE(good_tensor(grads[i], numel[i], types[i]));
  hipStream_t st = (hipStream_t)stream;
  double* part = (double*)workspace;
  int np = 0;
  for (int i = 0; i < count;) {
    Table tb;
    fill(tb, kTensors, kChunk, 0x7fffffff, numel, count, &i, [&](int k, int j) {
      tb.p[k] = const_cast<void*>(grads[j]);
      tb.type[k] = (unsigned char)types[j];
    });
    if (tb.count == 0) continue;
    const int blocks = tb.chunks < kNormBlocks ? tb.chunks : kNormBlocks;
    hipLaunchKernelGGL(norm_partial_kernel, dim3(blocks), dim3(256), 0, st, tb, part + np);
    MST_CHECK_LAUNCH();
    np += blocks;
  }
  hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(256), 0, st, part, np, norm);
  MST_CHECK_LAUNCH();
  return MST_OK;
}

int mst_grad_scale(void* const* grads, const int64_t* numel, const int32_t* types, int32_t count,
                   const float* norm, float max_norm, void* stream) {
  MST_REQUIRE(count >= 0 && norm && (count == 0 || (grads && numel && types)));
  MST_REQUIRE(max_norm >= 0.f);
  if (count == 0) return MST_OK;
  Range* r = new (std::nothrow) Range[count];
  MST_REQUIRE(r);
  int64_t n = 0;
  bool ok = true;
  for (int i = 0; i < count && ok; ++i) {
    ok = good_tensor(grads[i], numel[i], types[i]);
    const uintptr_t a = (uintptr_t)grads[i];
    if (numel[i] > 0) r[n++] = {a, a + (uintptr_t)numel[i] * size_of(types[i])};
  }
  ok = ok && !overlap(r, n);
  delete[] r;
  MST_REQUIRE(ok);
  for (int i = 0; i < count;) {
    Table tb;
    fill(tb, kTensors, kChunk, 0x7fffffff, numel, count, &i, [&](int k, int j) {
      tb.p[k] = grads[j];
      tb.type[k] = (unsigned char)types[j];
    });
    if (tb.count == 0) continue;
    hipLaunchKernelGGL(clip_scale_kernel, dim3(tb.chunks < kMaxChunks ? tb.chunks : kMaxChunks), dim3(256), 0,
                       (hipStream_t)stream, tb, norm, max_norm);
    MST_CHECK_LAUNCH();
  }
  return MST_OK;
}

int mst_adam_clip_f32(float* const* p, const float* const* g, float* const* m, float* const* v,
                      const int64_t* numel, int32_t count, const float* norm, float max_norm,
                      float lr_step, float b2, float one_minus_b1, float one_minus_b2, float eps,
                      float bc2_sqrt, const float* hyper, void* stream) {
  MST_REQUIRE(count >= 0 && norm && (count == 0 || (p && g && m && v && numel)));
  MST_REQUIRE(max_norm >= 0.f);
  if (count == 0) return MST_OK;
  Range* r = new (std::nothrow) Range[3 * (size_t)count];
  MST_REQUIRE(r);
  int64_t n = 0;
  bool ok = true;
  for (int i = 0; i < count && ok; ++i) {
    const void* all[4] = {p[i], m[i], v[i], g[i]};
    for (int k = 0; k < 4; ++k) {
      ok = ok && good_tensor(all[k], numel[i], MST_F32);
      const uintptr_t a = (uintptr_t)all[k];
      if (k < 3 && numel[i] > 0) r[n++] = {a, a + (uintptr_t)numel[i] * 4};
    }
  }
  ok = ok && !overlap(r, n);
  delete[] r;
  MST_REQUIRE(ok);
  const AdamK k = {lr_step, b2, one_minus_b1, one_minus_b2, eps, bc2_sqrt};
  for (int i = 0; i < count;) {
    AdamTable tb;
    fill(tb, kAdamTensors, kAdamChunk, kMaxChunks, numel, count, &i, [&](int q, int j) {
      tb.p[q] = p[j], tb.g[q] = g[j], tb.m[q] = m[j], tb.v[q] = v[j];
    });
    if (tb.count == 0) continue;
    hipLaunchKernelGGL(adam_clip_kernel, dim3(tb.chunks), dim3(256), 0, (hipStream_t)stream, tb, norm, max_norm, k, hyper);
    MST_CHECK_LAUNCH();
  }
  return MST_OK;
}

}  // extern "C"
