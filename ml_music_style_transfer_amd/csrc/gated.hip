// Gated linear recurrence over time (B, C, T), forward, backward and single frame.
//
//   a_t = sigmoid(gate_t)      h_t = a_t h_{t-1} + (1 - a_t) x_t       (t runs down when reversed)
// Frames at or past a clip's length are the identity map: the state passes, h = 0 there.
//
// A frame is the affine map h -> a h + b, b = (1 - a) x, and maps compose associatively:
// (a2, b2) after (a1, b1) = (a2 a1, a2 b1 + b2). A row (b, c) belongs to a group of W lanes, each
// lane to V consecutive frames: the lane composes its maps, the group scans the compositions with
// shuffles, and each lane then runs its frames from the state that enters them. W lanes x V frames
// are a tile; longer rows walk their tiles with the state in a register. Everything between the
// loads and the stores is 32-bit float.
//
// Backward: dh_t = gh_t + u_{t+1}, u_t = a_t dh_t (what frame t hands back) is the same kind of
// scan against the direction of time, u_t = a_t u_{t+1} + a_t gh_t;
//   dx_t = (1 - a_t) dh_t      dgate_t = dh_t (h_{t-1} - x_t) a_t (1 - a_t)      dh0 = u_0
// h_{t-1} is computed again from x, gate and the state that entered the tile (`carry`, kept by the
// forward): reading h back would cost another tensor and, in 16 bits, its rounding.
#include "common.h"

namespace {

constexpr int kV = 4;           // frames of a lane
constexpr int kTile = 64 * kV;  // frames of a whole wave: the step of `carry`

struct Args {
  const void *x, *gate;  // (B, C, T) by batch and channel strides, unit time stride
  long long xb, xc, gb, gc;
  const float* h0;     // (B, C), nullable
  const int32_t* len;  // (B), nullable
  void* h;             // (B, C, T) contiguous
  float* last;         // (B, C)
  float* carry;        // (B, C, tiles) state that enters a tile; unused with one tile
  // backward
  const void* gh;      // (B, C, T) contiguous, nullable
  const float* glast;  // (B, C), nullable
  void *dx, *dgate;    // (B, C, T) contiguous
  float* dh0;          // (B, C), nullable
  int32_t C, T, tiles;
  long long rows;
};

template <typename T> struct Vec;
template <> struct Vec<float> { typedef float t __attribute__((ext_vector_type(kV), aligned(4))); };
template <> struct Vec<__bf16> { typedef __bf16 t __attribute__((ext_vector_type(kV), aligned(2))); };
template <> struct Vec<_Float16> { typedef _Float16 t __attribute__((ext_vector_type(kV), aligned(2))); };

// frames [t, t + kV) of a row, zero from `end` on (nothing there is read)
template <typename T>
__device__ __forceinline__ void load(const T* row, int t, int end, float (&v)[kV]) {
  if (t + kV <= end) {
    const typename Vec<T>::t q = *reinterpret_cast<const typename Vec<T>::t*>(row + t);
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = (float)q[k];
  } else {
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = t + k < end ? (float)row[t + k] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store(T* row, int t, int end, const float (&v)[kV]) {
  if (t + kV <= end) {
    typename Vec<T>::t q;
#pragma unroll
    for (int k = 0; k < kV; ++k) q[k] = (T)v[k];
    *reinterpret_cast<typename Vec<T>::t*>(row + t) = q;
  } else {
#pragma unroll
    for (int k = 0; k < kV; ++k)
      if (t + k < end) row[t + k] = (T)v[k];
  }
}

// a = sigmoid(g) and c = 1 - a, each to its own relative precision (c is not formed from a)
__device__ __forceinline__ void gate_of(float g, float& a, float& c) {
  const float e = expf(-fabsf(g));
  const float r = 1.f / (1.f + e);
  a = g < 0.f ? e * r : r;
  c = g < 0.f ? r : e * r;
}

// Scan of the lanes' maps (A, H) over the W lanes of a row, in lane order or against it. In: a
// lane's own map. Out: the composition of the maps before it (the first lane: the identity) in
// (A, H), and of the whole row in (At, Ht).
template <int W, bool DOWN>
__device__ __forceinline__ void scan(float& A, float& H, float& At, float& Ht) {
  const int lane = threadIdx.x & (W - 1);
#pragma unroll
  for (int d = 1; d < W; d <<= 1) {
    const float a = DOWN ? __shfl_down(A, d, W) : __shfl_up(A, d, W);
    const float h = DOWN ? __shfl_down(H, d, W) : __shfl_up(H, d, W);
    if (DOWN ? lane + d < W : lane >= d) {
      H = fmaf(A, h, H);
      A *= a;
    }
  }
  At = __shfl(A, DOWN ? 0 : W - 1, W);
  Ht = __shfl(H, DOWN ? 0 : W - 1, W);
  A = DOWN ? __shfl_down(A, 1, W) : __shfl_up(A, 1, W);
  H = DOWN ? __shfl_down(H, 1, W) : __shfl_up(H, 1, W);
  if (lane == (DOWN ? W - 1 : 0)) A = 1.f, H = 0.f;
}

__device__ __forceinline__ int row_len(const Args& p, long long b) {
  if (!p.len) return p.T;
  const int n = p.len[b];
  return n < 0 ? 0 : n < p.T ? n : p.T;
}

template <typename T, int W, bool REV>
__global__ __launch_bounds__(256) void gated_fwd_kernel(const Args p) {
  const long long row = (blockIdx.x * 256ll + threadIdx.x) / W;
  if (row >= p.rows) return;
  const int lane = threadIdx.x & (W - 1);
  const long long b = row / p.C, c = row % p.C;
  const T* x = (const T*)p.x + b * p.xb + c * p.xc;
  const T* g = (const T*)p.gate + b * p.gb + c * p.gc;
  T* h = (T*)p.h + row * p.T;
  const int len = row_len(p, b);
  float s = p.h0 ? p.h0[row] : 0.f;
  for (int i = 0; i < p.tiles; ++i) {
    const int tile = REV ? p.tiles - 1 - i : i;
    const int t = tile * W * kV + lane * kV;
    if (p.tiles > 1 && lane == 0) p.carry[row * p.tiles + tile] = s;
    float xv[kV], gv[kV], a[kV];
    load(x, t, len, xv);
    load(g, t, len, gv);
    float A = 1.f, H = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? kV - 1 - q : q;
      float cc;
      gate_of(gv[k], a[k], cc);
      if (t + k >= len) a[k] = 1.f, cc = 0.f;
      xv[k] *= cc;
      H = fmaf(a[k], H, xv[k]);
      A *= a[k];
    }
    scan<W, REV>(A, H, At, Ht);
    float e = fmaf(A, s, H);
    s = fmaf(At, s, Ht);
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? kV - 1 - q : q;
      e = fmaf(a[k], e, xv[k]);
      xv[k] = t + k < len ? e : 0.f;
    }
    store(h, t, p.T, xv);
  }
  if (lane == 0) p.last[row] = s;
}

template <typename T, int W, bool REV>
__global__ __launch_bounds__(256) void gated_bwd_kernel(const Args p) {
  const long long row = (blockIdx.x * 256ll + threadIdx.x) / W;
  if (row >= p.rows) return;
  const int lane = threadIdx.x & (W - 1);
  const long long b = row / p.C, c = row % p.C;
  const T* x = (const T*)p.x + b * p.xb + c * p.xc;
  const T* g = (const T*)p.gate + b * p.gb + c * p.gc;
  const T* gh = p.gh ? (const T*)p.gh + row * p.T : nullptr;
  const int len = row_len(p, b);
  const float h0 = p.h0 ? p.h0[row] : 0.f;
  float s = p.glast ? p.glast[row] : 0.f;
  for (int i = 0; i < p.tiles; ++i) {
    const int tile = REV ? i : p.tiles - 1 - i;
    const int t = tile * W * kV + lane * kV;
    const float in = p.tiles > 1 ? p.carry[row * p.tiles + tile] : h0;
    float xv[kV], gv[kV], dv[kV], a[kV], cc[kV];
    load(x, t, len, xv);
    load(g, t, len, gv);
    load(gh ? gh : x, t, gh ? len : 0, dv);
    float A = 1.f, H = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? kV - 1 - q : q;
      gate_of(gv[k], a[k], cc[k]);
      if (t + k >= len) a[k] = 1.f, cc[k] = 0.f;
      H = fmaf(a[k], H, cc[k] * xv[k]);
      A *= a[k];
    }
    float U = 0.f, Ua = A;
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? q : kV - 1 - q;
      U = a[k] * (dv[k] + U);
    }
    scan<W, REV>(A, H, At, Ht);
    float e = fmaf(A, in, H);  // the state before the lane's first frame
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? kV - 1 - q : q;
      gv[k] = e - xv[k];
      e = fmaf(a[k], e, cc[k] * xv[k]);
    }
    scan<W, !REV>(Ua, U, At, Ht);
    float u = fmaf(Ua, s, U);  // what the frame after the lane's last hands back
    s = fmaf(At, s, Ht);
#pragma unroll
    for (int q = 0; q < kV; ++q) {
      const int k = REV ? q : kV - 1 - q;
      const float d = dv[k] + u;
      u = a[k] * d;
      const bool live = t + k < len;
      xv[k] = live ? cc[k] * d : 0.f;
      gv[k] = live ? u * cc[k] * gv[k] : 0.f;
    }
    store((T*)p.dx + row * p.T, t, p.T, xv);
    store((T*)p.dgate + row * p.T, t, p.T, gv);
  }
  if (p.dh0 && lane == 0) p.dh0[row] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void gated_step_kernel(const T* __restrict__ x, long long xb,
                                                         const T* __restrict__ gate, long long gb,
                                                         float* __restrict__ state, T* __restrict__ h,
                                                         int C, long long n) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long b = i / C, c = i % C;
  float a, cc;
  gate_of((float)gate[b * gb + c], a, cc);
  const float s = fmaf(a, state[i], cc * (float)x[b * xb + c]);
  state[i] = s;
  h[i] = (T)s;
}

int tiles_of(int32_t T) { return (T + kTile - 1) / kTile; }

// lanes of a row: the fewest that hold it in one tile
int lanes_of(int32_t T) {
  int w = 4;
  while (w < 64 && w * kV < T) w *= 2;
  return w;
}

template <typename T, bool REV, bool BWD>
void launch_w(const Args& p, hipStream_t st) {
  const int w = lanes_of(p.T);
  const dim3 grid((unsigned)((p.rows * w + 255) / 256));
#define MST_GATED(W_)                                                                        \
  do {                                                                                       \
    if (BWD) hipLaunchKernelGGL((gated_bwd_kernel<T, W_, REV>), grid, dim3(256), 0, st, p);  \
    else hipLaunchKernelGGL((gated_fwd_kernel<T, W_, REV>), grid, dim3(256), 0, st, p);      \
  } while (0)
  if (w == 4) MST_GATED(4);
  else if (w == 8) MST_GATED(8);
  else if (w == 16) MST_GATED(16);
  else if (w == 32) MST_GATED(32);
  else MST_GATED(64);
#undef MST_GATED
}

template <bool BWD>
int launch(const Args& p, int type, int reverse, hipStream_t st) {
  if (type == MST_F32) reverse ? launch_w<float, true, BWD>(p, st) : launch_w<float, false, BWD>(p, st);
  else if (type == MST_BF16) reverse ? launch_w<__bf16, true, BWD>(p, st) : launch_w<__bf16, false, BWD>(p, st);
  else reverse ? launch_w<_Float16, true, BWD>(p, st) : launch_w<_Float16, false, BWD>(p, st);
  MST_CHECK_LAUNCH();
  return MST_OK;
}

bool good_shape(int32_t type, int32_t B, int32_t C, int32_t T) {
  return type >= MST_F32 && type <= MST_F16 && B > 0 && C > 0 && T > 0 &&
         (long long)B * C <= (1ll << 31) && T <= 0x7fffffff - kTile;
}

}  // namespace

extern "C" {

int32_t mst_gated_tiles(int32_t T) { return T > kTile ? tiles_of(T) : 0; }

int mst_gated_fwd(int32_t type, const void* x, int64_t xb, int64_t xc, const void* gate, int64_t gb,
                  int64_t gc, const float* h0, const int32_t* lengths, int32_t B, int32_t C, int32_t T,
                  int32_t reverse, void* h, float* last, float* carry, void* stream) {
  MST_REQUIRE(good_shape(type, B, C, T) && x && gate && h && last);
  MST_REQUIRE(T <= kTile || carry);
  Args p = {};
  p.x = x, p.xb = xb, p.xc = xc, p.gate = gate, p.gb = gb, p.gc = gc;
  p.h0 = h0, p.len = lengths, p.h = h, p.last = last, p.carry = carry;
  p.C = C, p.T = T, p.tiles = tiles_of(T), p.rows = (long long)B * C;
  return launch<false>(p, type, reverse, (hipStream_t)stream);
}

int mst_gated_bwd(int32_t type, const void* x, int64_t xb, int64_t xc, const void* gate, int64_t gb,
                  int64_t gc, const float* h0, const int32_t* lengths, const float* carry,
                  const void* gh, const float* glast, int32_t B, int32_t C, int32_t T, int32_t reverse,
                  void* dx, void* dgate, float* dh0, void* stream) {
  MST_REQUIRE(good_shape(type, B, C, T) && x && gate && dx && dgate);
  MST_REQUIRE(T <= kTile || carry);
  Args p = {};
  p.x = x, p.xb = xb, p.xc = xc, p.gate = gate, p.gb = gb, p.gc = gc;
  p.h0 = h0, p.len = lengths, p.carry = const_cast<float*>(carry);
  p.gh = gh, p.glast = glast, p.dx = dx, p.dgate = dgate, p.dh0 = dh0;
  p.C = C, p.T = T, p.tiles = tiles_of(T), p.rows = (long long)B * C;
  return launch<true>(p, type, reverse, (hipStream_t)stream);
}

int mst_gated_step(int32_t type, const void* x, int64_t xb, const void* gate, int64_t gb, int32_t B,
                   int32_t C, float* state, void* h, void* stream) {
  MST_REQUIRE(good_shape(type, B, C, 1) && x && gate && state && h);
  const long long n = (long long)B * C;
  const dim3 grid((unsigned)((n + 255) / 256));
  hipStream_t st = (hipStream_t)stream;
  if (type == MST_F32)
    hipLaunchKernelGGL(gated_step_kernel<float>, grid, dim3(256), 0, st, (const float*)x, xb,
                       (const float*)gate, gb, state, (float*)h, C, n);
  else if (type == MST_BF16)
    hipLaunchKernelGGL(gated_step_kernel<__bf16>, grid, dim3(256), 0, st, (const __bf16*)x, xb,
                       (const __bf16*)gate, gb, state, (__bf16*)h, C, n);
  else
    hipLaunchKernelGGL(gated_step_kernel<_Float16>, grid, dim3(256), 0, st, (const _Float16*)x, xb,
                       (const _Float16*)gate, gb, state, (_Float16*)h, C, n);
  MST_CHECK_LAUNCH();
  return MST_OK;
}

}  // extern "C"
