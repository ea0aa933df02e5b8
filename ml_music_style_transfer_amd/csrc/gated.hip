// Gated linear recurrence over time (B, C, T), forward, backward and single frame.
//
//   a_t = sigmoid(gate_t)      h_t = a_t h_{t-1} + (1 - a_t) x_t       (t runs down when reversed)
// Frames at or past a clip's length are the identity map: the state passes, h = 0 there.
//
// A frame is the affine map h -> a h + b, b = (1 - a) x, and maps compose associatively:
// (a2, b2) after (a1, b1) = (a2 a1, a2 b1 + b2). A row (b, c) belongs to a group of W lanes, each
// lane to V = 8 consecutive frames: the lane composes its maps, the group scans the compositions
// (DPP row shifts: no LDS for 16 lanes, a scan costs about 4 VALU a level), and each lane then runs
// its frames from the state that enters them. W lanes x V frames are a tile; longer rows walk their
// tiles with the state in a register and the next tile's loads in flight. Everything between the
// loads and the stores is 32-bit float.
//
// Backward: dh_t = gh_t + u_{t+1}, u_t = a_t dh_t (what frame t hands back) is the same kind of
// scan against the direction of time, u_t = a_t u_{t+1} + a_t gh_t;
//   dx_t = (1 - a_t) dh_t      dgate_t = dh_t (h_{t-1} - x_t) a_t (1 - a_t)      dh0 = u_0
// h_{t-1} is computed again from x, gate and the state that entered the tile (`carry`, kept by the
// forward): reading h back would cost another tensor and, in 16 bits, its rounding.
#include "common.h"

namespace {

constexpr int V = 8;           // frames of a lane
constexpr int kTile = 64 * V;  // frames of a whole wave: the step of `carry`

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
  uint32_t rows;
};

// P elements are 16 bytes, at the element's own alignment (rows may start anywhere)
template <typename T> struct Piece;
template <> struct Piece<float> { typedef float t __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Piece<__bf16> { typedef __bf16 t __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Piece<_Float16> { typedef _Float16 t __attribute__((ext_vector_type(8), aligned(2))); };

// a lane's V frames as they lie in memory: converted after the next tile's loads are under way
template <typename T> struct Raw {
  static constexpr int P = 16 / sizeof(T), N = V / P;
  typename Piece<T>::t q[N];

  // frames [t, t + V) of a row; those from `end` on hold anything (nothing there is read)
  __device__ __forceinline__ void load(const T* row, int t, int end) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = t + i * P;
      if (s + P <= end) {
        q[i] = *reinterpret_cast<const typename Piece<T>::t*>(row + s);
      } else if (s < end) {
#pragma unroll
        for (int k = 0; k < P; ++k) q[i][k] = row[min(s + k, end - 1)];
      }
    }
  }
  __device__ __forceinline__ float operator[](int k) const { return (float)q[k / P][k % P]; }
};

template <typename T>
__device__ __forceinline__ void store(T* row, int t, int end, const float (&v)[V]) {
  constexpr int P = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < V / P; ++i) {
    const int s = t + i * P;
    if (s + P <= end) {
      typename Piece<T>::t q;
#pragma unroll
      for (int k = 0; k < P; ++k) q[k] = (T)v[i * P + k];
      *reinterpret_cast<typename Piece<T>::t*>(row + s) = q;
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k)
        if (s + k < end) row[s + k] = (T)v[i * P + k];
    }
  }
}

// a = sigmoid(g) and c = 1 - a, each to its own relative precision (c is not formed from a).
// e^-m = 2^t e^(-m - t ln 2) with t = -m log2(e) rounded: the second factor is 1 + a rounding's
// size. Past 150 the first is 0, as it is for infinite g; a g that is not a number stays none.
__device__ __forceinline__ void gate_of(float g, float& a, float& c) {
  const float m = fabsf(g) > 150.f ? 150.f : fabsf(g);
  const float t = m * -1.44269504f;
  float e = __builtin_amdgcn_exp2f(t);
  e = fmaf(e, fmaf(t, -0.693147181f, -m), e);
  const float d = 1.f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(r, fmaf(-d, r, 1.f), r);  // one Newton step: the quotient to half a step
  const float er = e * r;
  a = g < 0.f ? er : r;
  c = g < 0.f ? r : er;
}

// lane's value from the lane that the DPP control names, `old` where it names none
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float old, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old),
                                                              __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
constexpr int kRowShl = 0x100, kRowShr = 0x110, kWaveShl1 = 0x130, kWaveShr1 = 0x138, kBcast15 = 0x142,
              kBcast31 = 0x143;

// One level of the scan: every lane takes the composition of the lanes D before it (after it with
// DOWN) in its group of W, the identity where there are none.
template <int W, bool DOWN, int D>
__device__ __forceinline__ void level(float& A, float& H) {
  const int lane = threadIdx.x & 63;
  float a, h;
  if constexpr (D < 16) {
    a = dpp<(DOWN ? kRowShl : kRowShr) + D>(1.f, A);
    h = dpp<(DOWN ? kRowShl : kRowShr) + D>(0.f, H);
    if constexpr (W < 16) {  // a row of 16 lanes holds several groups
      const bool in = DOWN ? (lane & (W - 1)) + D < W : (lane & (W - 1)) >= D;
      a = in ? a : 1.f;
      h = in ? h : 0.f;
    }
  } else if constexpr (!DOWN) {  // the last lane of the 16 (32) lanes before, for every second 16 (32)
    a = dpp<D == 16 ? kBcast15 : kBcast31, D == 16 ? 0xa : 0xc>(1.f, A);
    h = dpp<D == 16 ? kBcast15 : kBcast31, D == 16 ? 0xa : 0xc>(0.f, H);
  } else {  // the first lane of the 16 (32) lanes after
    const int from = (lane & ~(D - 1)) + D;
    const bool in = (lane & D) == 0;
    a = __shfl(A, from & 63, 64);
    h = __shfl(H, from & 63, 64);
    a = in ? a : 1.f;
    h = in ? h : 0.f;
  }
  H = fmaf(A, h, H);
  A *= a;
}

// Scan of the lanes' maps (A, H) over the W lanes of a row, in lane order or against it. In: a
// lane's own map. Out: the composition of the maps before it (the first lane: the identity); for
// a whole wave also that of the row in (At, Ht).
template <int W, bool DOWN>
__device__ __forceinline__ void scan(float& A, float& H, float& At, float& Ht) {
  level<W, DOWN, 1>(A, H);
  level<W, DOWN, 2>(A, H);
  if constexpr (W > 4) level<W, DOWN, 4>(A, H);
  if constexpr (W > 8) level<W, DOWN, 8>(A, H);
  if constexpr (W > 16) level<W, DOWN, 16>(A, H);
  if constexpr (W > 32) {
    level<W, DOWN, 32>(A, H);
    At = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, A), DOWN ? 0 : 63));
    Ht = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, H), DOWN ? 0 : 63));
  }
  A = dpp<DOWN ? kWaveShl1 : kWaveShr1>(1.f, A);
  H = dpp<DOWN ? kWaveShl1 : kWaveShr1>(0.f, H);
  if constexpr (W < 64)
    if ((threadIdx.x & (W - 1)) == (DOWN ? W - 1 : 0)) A = 1.f, H = 0.f;
}

// the rows of x and gate, and the clip's length, of row `row`
template <typename T> struct Row {
  const T *x, *g;
  int len;
  __device__ __forceinline__ Row(const Args& p, uint32_t row) {
    const uint32_t b = row / (uint32_t)p.C, c = row % (uint32_t)p.C;
    x = (const T*)p.x + b * p.xb + c * p.xc;
    g = (const T*)p.gate + b * p.gb + c * p.gc;
    const int n = p.len ? p.len[b] : p.T;
    len = n < 0 ? 0 : n < p.T ? n : p.T;
  }
};

// row of the calling lane's group; the same scalar for the whole wave when a group is one
template <int W>
__device__ __forceinline__ uint32_t group_id() {
  const uint32_t i = blockIdx.x * (256u / W) + threadIdx.x / W;
  return W == 64 ? __builtin_amdgcn_readfirstlane(i) : i;
}

template <typename T, int W, bool REV>
__global__ __launch_bounds__(256) void gated_fwd_kernel(const Args p) {
  const uint32_t row = group_id<W>();
  if (row >= p.rows) return;
  const int lane = threadIdx.x & (W - 1);
  const Row<T> r(p, row);
  T* h = (T*)p.h + (long long)row * p.T;
  float s = p.h0 ? p.h0[row] : 0.f;
  int t = (REV ? p.tiles - 1 : 0) * (W * V) + lane * V;
  Raw<T> xr, gr;
  xr.load(r.x, t, r.len);
  gr.load(r.g, t, r.len);
  for (int i = 0; i < p.tiles; ++i) {
    if (W == 64 && p.tiles > 1 && lane == 0)
      p.carry[(long long)row * p.tiles + (REV ? p.tiles - 1 - i : i)] = s;
    float b[V], a[V], c[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      b[k] = xr[k];
      gate_of(gr[k], a[k], c[k]);
    }
    const int now = t;
    if (W == 64 && i + 1 < p.tiles) {
      t += REV ? -kTile : kTile;
      xr.load(r.x, t, r.len);
      gr.load(r.g, t, r.len);
    }
    if (now + V > r.len) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (now + k >= r.len) a[k] = 1.f, b[k] = c[k] = 0.f;
    }
    float A = 1.f, H = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q;
      b[k] *= c[k];
      H = fmaf(a[k], H, b[k]);
      A *= a[k];
    }
    scan<W, REV>(A, H, At, Ht);
    float e = fmaf(A, s, H);
    if (W == 64) s = fmaf(At, s, Ht);
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q;
      e = fmaf(a[k], e, b[k]);
      b[k] = e;
    }
    if (W < 64) s = e;
    if (now + V > r.len) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (now + k >= r.len) b[k] = 0.f;
    }
    store(h, now, p.T, b);
  }
  if (lane == (W == 64 || REV ? 0 : W - 1)) p.last[row] = s;
}

template <typename T, int W, bool REV>
__global__ __launch_bounds__(256) void gated_bwd_kernel(const Args p) {
  const uint32_t row = group_id<W>();
  if (row >= p.rows) return;
  const int lane = threadIdx.x & (W - 1);
  const Row<T> r(p, row);
  const T* gh = p.gh ? (const T*)p.gh + (long long)row * p.T : r.x;
  const int ghlen = p.gh ? r.len : 0;
  float s = p.glast ? p.glast[row] : 0.f;
  const float h0 = p.h0 ? p.h0[row] : 0.f;
  int t = (REV ? 0 : p.tiles - 1) * (W * V) + lane * V;
  Raw<T> xr, gr, dr;
  xr.load(r.x, t, r.len);
  gr.load(r.g, t, r.len);
  dr.load(gh, t, ghlen);
  for (int i = 0; i < p.tiles; ++i) {
    const float in = W == 64 && p.tiles > 1
                         ? p.carry[(long long)row * p.tiles + (REV ? i : p.tiles - 1 - i)] : h0;
    float x[V], d[V], a[V], c[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      x[k] = xr[k];
      d[k] = dr[k];
      gate_of(gr[k], a[k], c[k]);
    }
    const int now = t;
    if (W == 64 && i + 1 < p.tiles) {
      t += REV ? kTile : -kTile;
      xr.load(r.x, t, r.len);
      gr.load(r.g, t, r.len);
      dr.load(gh, t, ghlen);
    }
    if (now + V > r.len) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (now + k >= r.len) a[k] = 1.f, c[k] = x[k] = d[k] = 0.f;
    }
    if (!p.gh) {
#pragma unroll
      for (int k = 0; k < V; ++k) d[k] = 0.f;
    }
    float A = 1.f, H = 0.f, U = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q, j = V - 1 - k;
      H = fmaf(a[k], H, c[k] * x[k]);
      A *= a[k];
      U = a[j] * (d[j] + U);
    }
    float Ua = A;
    scan<W, REV>(A, H, At, Ht);
    scan<W, !REV>(Ua, U, At, Ht);
    float e = fmaf(A, in, H);   // the state before the lane's first frame
    float u = fmaf(Ua, s, U);   // what the frame after the lane's last hands back
    if (W == 64) s = fmaf(At, s, Ht);
    float diff[V];
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q;
      diff[k] = e - x[k];
      e = fmaf(a[k], e, c[k] * x[k]);
    }
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? q : V - 1 - q;
      const float dh = d[k] + u;
      u = a[k] * dh;
      x[k] = c[k] * dh;
      diff[k] *= u * c[k];
    }
    if (W < 64) s = u;
    if (now + V > r.len) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (now + k >= r.len) x[k] = diff[k] = 0.f;
    }
    store((T*)p.dx + (long long)row * p.T, now, p.T, x);
    store((T*)p.dgate + (long long)row * p.T, now, p.T, diff);
  }
  if (p.dh0 && lane == (W == 64 || !REV ? 0 : W - 1)) p.dh0[row] = s;
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
  while (w < 64 && w * V < T) w *= 2;
  return w;
}

template <typename T, bool REV, bool BWD>
void launch_w(const Args& p, hipStream_t st) {
  const int w = lanes_of(p.T);
  const dim3 grid((unsigned)(((long long)p.rows * w + 255) / 256));
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
         (long long)B * C < (1ll << 31) && T <= 0x7fffffff - kTile;
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
  p.C = C, p.T = T, p.tiles = tiles_of(T), p.rows = (uint32_t)B * (uint32_t)C;
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
  p.C = C, p.T = T, p.tiles = tiles_of(T), p.rows = (uint32_t)B * (uint32_t)C;
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
