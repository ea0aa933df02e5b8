// Gated linear recurrence over time (B, C, T), forward, backward and single frame.
//
//   a_t = sigmoid(gate_t)      h_t = a_t h_{t-1} + (1 - a_t) x_t       (t runs down when reversed)
// Frames at or past a clip's length are the identity map: the state passes, h = 0 there.
//
// A frame is the affine map h -> a h + b, b = (1 - a) x, and maps compose associatively:
// (a2, b2) after (a1, b1) = (a2 a1, a2 b1 + b2). A row (b, c) belongs to a group of W lanes, each
// lane to V = 8 consecutive frames: the lane composes its maps, the group scans the compositions
// (DPP row shifts: two instructions a level and no LDS within 16 lanes), and each lane then runs
// its frames from the state that enters them. W lanes x V frames are a tile; longer rows walk their
// tiles with the state in a register and the next tile's loads in flight. Everything between the
// loads and the stores is 32-bit float.
//
// Backward: dh_t = gh_t + u_{t+1}, u_t = a_t dh_t (what frame t hands back) is the same kind of
// scan against the direction of time, u_t = a_t u_{t+1} + a_t gh_t;
//   dx_t = (1 - a_t) dh_t      dgate_t = dh_t (h_{t-1} - x_t) a_t (1 - a_t)      dh0 = u_0
// h_{t-1} is computed again from x, gate and the state that entered the tile (`carry`, kept by the
// forward): reading h back would cost another tensor and, in 16 bits, its rounding.
//
// Bound by HBM in float32: (32, 1024, 252) takes 17 us forward and 27 us backward, 5.9 and 6.2 TB/s
// of the 3 and 5 tensors that have to move. In 16 bits also by the vector unit's issue: a frame
// costs some 28 instructions forward and 43 backward (14 of them its gate; two more in float32), and
// (16, 4096, 860) in bfloat16 takes 62 and 107 us, 5.5 and 5.3 TB/s. With padded clips, whose loads stop at
// their lengths but whose frames are all computed, it takes nearly as long (61 and 101 us; 93 % and 84 % of the
// issue slots, 3.8 and 4.0 TB/s of what has to move): issue alone. Rows of an odd number of 16-bit
// frames, which start off any alignment, are the slowest ((64, 8192, 63) backward 83 us, 4.0 TB/s).
#include "common.h"

namespace {

constexpr int kV = 8;           // frames of a lane
// 16-bit rows that 16 frames a lane fit into one tile: (16, 4096, 860) bfloat16, two tiles -> one, 69 + 109
// -> 63 + 107 us; not float32 ((16, 2048, 860): 63 + 112 -> 71 + 122, its loads no longer fill lines)
constexpr int kWide = 16;
constexpr int kTile = 64 * kV;  // frames of a wave in rows of several tiles: the step of `carry`

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
  // A long axis with few rows: `segs` waves a row, each `span` tiles. Their maps, in the order of
  // the pass, are composed first (maps, (rows, segs)); each wave enters with those before it.
  float2* maps;
  int32_t segs, span;
  int32_t C, T, tiles;
  uint32_t rows;
};

// P elements are 16 bytes, at the element's own alignment (rows may start anywhere)
template <typename T> struct Piece;
template <> struct Piece<float> { typedef float t __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Piece<__bf16> { typedef __bf16 t __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Piece<_Float16> { typedef _Float16 t __attribute__((ext_vector_type(8), aligned(2))); };

// A lane's V frames as they lie in memory: converted after the next tile's loads are under way.
// Loads are free of branches (at a join the compiler would wait for their data): a piece that ends
// past `end` reads the last 16 bytes before it, and settle() moves what belongs to the lane down.
// Frames past the clip hold anything. `end` is the clip's length, or P in a shorter clip: the row
// has T >= P frames. SHORT: rows of T < P frames, read frame by frame.
template <typename T, int V, bool SHORT> struct Raw {
  static constexpr int P = 16 / sizeof(T), N = V / P;
  typename Piece<T>::t q[N];

  __device__ __forceinline__ void load(const T* row, int t, int end) {
    if constexpr (SHORT) {
#pragma unroll
      for (int k = 0; k < P; ++k) q[0][k] = row[min(t + k, end - 1)];
#pragma unroll
      for (int i = 1; i < N; ++i) q[i] = q[0];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        q[i] = *reinterpret_cast<const typename Piece<T>::t*>(row + max(min(t + i * P, end - P), 0));
    }
  }
  __device__ __forceinline__ void settle(int t, int end) {
    if constexpr (!SHORT) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int n = t + i * P - (end - P);
        if (0 < n && n < P) down(q[i], n);
      }
    }
  }
  // q[k] <- q[k + n], 0 < n < P, by the bits of n (as words where n allows)
  static __device__ __forceinline__ void down(typename Piece<T>::t& q, int n) {
    if constexpr (P == 8) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      u32x4 w = __builtin_bit_cast(u32x4, q);
      if (n & 4) w[0] = w[2], w[1] = w[3];
      if (n & 2) w[0] = w[1], w[1] = w[2], w[2] = w[3];
      if (n & 1) {
#pragma unroll
        for (int k = 0; k < 3; ++k) w[k] = __builtin_amdgcn_alignbit(w[k + 1], w[k], 16);
        w[3] >>= 16;
      }
      q = __builtin_bit_cast(typename Piece<T>::t, w);
    } else {
      if (n & 2) q[0] = q[2], q[1] = q[3];
      if (n & 1) q[0] = q[1], q[1] = q[2], q[2] = q[3];
    }
  }
  __device__ __forceinline__ float operator[](int k) const { return (float)q[k / P][k % P]; }
};

template <typename T, int V>
__device__ __forceinline__ void store(T* row, int t, int end, const float (&v)[V]) {
  constexpr int P = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < V / P; ++i) {
    const int s = t + i * P;
    if (s >= end) break;
    typename Piece<T>::t q;
#pragma unroll
    for (int k = 0; k < P; ++k) q[k] = (T)v[i * P + k];
    if (s + P <= end) {
      *reinterpret_cast<typename Piece<T>::t*>(row + s) = q;
    } else {  // the row's end, by the bits of what is left
      int n = end - s;
      T* to = row + s;
      if constexpr (P == 8) {
        if (n & 4) {
          typedef T half __attribute__((ext_vector_type(4), aligned(sizeof(T))));
          *reinterpret_cast<half*>(to) = half{q[0], q[1], q[2], q[3]};
          q[0] = q[4], q[1] = q[5], q[2] = q[6];
          to += 4;
        }
      }
      if (n & 2) {
        to[0] = q[0], to[1] = q[1];
        q[0] = q[2];
        to += 2;
      }
      if (n & 1) to[0] = q[0];
    }
  }
}

// a = sigmoid(g) and c = 1 - a, each to its own relative precision (c is not formed from a).
// e^-|g| = 2^t e^(-|g| - t ln 2) with t = -|g| log2(e) rounded: the second factor is 1 + a rounding's
// size (taken into [-1, 1], since an infinite g makes its exponent no number where 2^t is zero; of a
// g that is no number 2^t is none either). e keeps the hardware exponential's error of one place and its
// correction's half (worst measured: 4.4 x 2^-24 of e). The quotient is the hardware's, to its last place,
// and for float32 tensors brought to the nearest by a step of Newton's: a on gates of 3 to 16 is off by
// 1.50 x 2^-24 at worst, 1.82 without; (32, 1024, 252) takes 17.2 + 27.2 us, 17.1 + 27.1 without. 16-bit
// kernels have no instruction to spare, and round what they store to 2^-8 or 2^-11.
template <typename T>
__device__ __forceinline__ void gate_of(float g, float& a, float& c) {
  const float t = fabsf(g) * -1.44269504f;
  float e = __builtin_amdgcn_exp2f(t);
  e = fmaf(e, __builtin_amdgcn_fmed3f(fmaf(t, -0.693147181f, -fabsf(g)), -1.f, 1.f), e);
  float r = __builtin_amdgcn_rcpf(1.f + e);
  if constexpr (sizeof(T) == 4) r = fmaf(fmaf(-(1.f + e), r, 1.f), r, r);
  const float er = e * r;
  a = g < 0.f ? er : r;
  c = g < 0.f ? r : er;
}

// frames from `n` on become the identity: an infinite gate holds the state, and x adds nothing
template <int V>
__device__ __forceinline__ void hold(int n, float (&g)[V], float (&x)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    g[k] = k < n ? g[k] : __builtin_inff();
    x[k] = k < n ? x[k] : 0.f;
  }
}
template <int V>
__device__ __forceinline__ void clear(int n, float (&v)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = k < n ? v[k] : 0.f;
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
  if constexpr (D < 16) {  // several groups in a row of 16 lanes
    const bool in = DOWN ? (lane & (W - 1)) + D < W : (lane & (W - 1)) >= D;
    a = dpp<(DOWN ? kRowShl : kRowShr) + D>(1.f, A);
    h = dpp<(DOWN ? kRowShl : kRowShr) + D>(0.f, H);
    a = in ? a : 1.f;
    h = in ? h : 0.f;
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

// Levels 1 to 8 as fused DPP instructions, for groups of 16 lanes or more: a lane whose source is
// outside its row of 16 is not written, which is the identity. A DPP operand may be read two
// instructions after it is written at the earliest: two independent scans keep each other's
// distance, one alone waits.
#define MST_FMAC(H, A, C) "v_fmac_f32_dpp " H ", " H ", " A " " C " row_mask:0xf bank_mask:0xf\n\t"
#define MST_MUL(A, C) "v_mul_f32_dpp " A ", " A ", " A " " C " row_mask:0xf bank_mask:0xf\n\t"
#define MST_ONE(C) MST_FMAC("%0", "%1", C) MST_MUL("%1", C) "s_nop 1\n\t"
#define MST_TWO(C, D) MST_FMAC("%0", "%1", C) MST_MUL("%1", C) MST_FMAC("%2", "%3", D) MST_MUL("%3", D)
template <bool DOWN>
__device__ __forceinline__ void levels16(float& A, float& H) {
  if constexpr (DOWN)
    asm volatile("s_nop 1\n\t" MST_ONE("row_shl:1") MST_ONE("row_shl:2") MST_ONE("row_shl:4") MST_ONE("row_shl:8")
                 : "+v"(H), "+v"(A));
  else
    asm volatile("s_nop 1\n\t" MST_ONE("row_shr:1") MST_ONE("row_shr:2") MST_ONE("row_shr:4") MST_ONE("row_shr:8")
                 : "+v"(H), "+v"(A));
}
// (A, H) in lane order and (B, K) against it
__device__ __forceinline__ void levels16_two(float& A, float& H, float& B, float& K) {
  asm volatile("s_nop 1\n\t" MST_TWO("row_shr:1", "row_shl:1") MST_TWO("row_shr:2", "row_shl:2")
               MST_TWO("row_shr:4", "row_shl:4") MST_TWO("row_shr:8", "row_shl:8") "s_nop 1"
               : "+v"(H), "+v"(A), "+v"(K), "+v"(B));
}
#undef MST_FMAC
#undef MST_MUL
#undef MST_ONE
#undef MST_TWO

// The levels above 8, the row's total and the step from "up to this lane" to "before it".
template <int W, bool DOWN>
__device__ __forceinline__ void finish_scan(float& A, float& H, float& At, float& Ht) {
  if constexpr (W > 16) level<W, DOWN, 16>(A, H);
  if constexpr (W > 32) {
    level<W, DOWN, 32>(A, H);
    At = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, A), DOWN ? 0 : 63));
    Ht = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, H), DOWN ? 0 : 63));
  }
  if constexpr (W > 1) {
    A = dpp<DOWN ? kWaveShl1 : kWaveShr1>(1.f, A);
    H = dpp<DOWN ? kWaveShl1 : kWaveShr1>(0.f, H);
  }
  if constexpr (W < 64)
    if ((threadIdx.x & (W - 1)) == (DOWN ? W - 1 : 0)) A = 1.f, H = 0.f;
}

// Scan of the lanes' maps (A, H) over the W lanes of a row, in lane order or against it. In: a
// lane's own map. Out: the composition of the maps before it (the first lane: the identity); for
// a whole wave also that of the row in (At, Ht).
template <int W, bool DOWN>
__device__ __forceinline__ void scan(float& A, float& H, float& At, float& Ht) {
  if constexpr (W >= 16) {
    levels16<DOWN>(A, H);
  } else {
    if constexpr (W > 1) level<W, DOWN, 1>(A, H);
    if constexpr (W > 2) level<W, DOWN, 2>(A, H);
    if constexpr (W > 4) level<W, DOWN, 4>(A, H);
  }
  finish_scan<W, DOWN>(A, H, At, Ht);
}

// scan of (A, H) with DOWN and of (B, K) against it; (Bt, Kt) is the second's total
template <int W, bool DOWN>
__device__ __forceinline__ void scan_two(float& A, float& H, float& B, float& K, float& Bt, float& Kt) {
  float At, Ht;
  if constexpr (W >= 16) {
    if constexpr (DOWN) levels16_two(B, K, A, H);
    else levels16_two(A, H, B, K);
    finish_scan<W, DOWN>(A, H, At, Ht);
    finish_scan<W, !DOWN>(B, K, Bt, Kt);
  } else {
    scan<W, DOWN>(A, H, At, Ht);
    scan<W, !DOWN>(B, K, Bt, Kt);
  }
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

// The state that enters segment `seg`: `s` through the maps of the segments before it.
__device__ __forceinline__ float enter(const Args& p, uint32_t row, int seg, float s) {
  const float2* m = p.maps + (long long)row * p.segs;
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < seg; i += 64) {
    float2 v = make_float2(1.f, 0.f);
    if (i + lane < seg) v = m[i + lane];
    float At, Ht;
    scan<64, false>(v.x, v.y, At, Ht);
    s = fmaf(At, s, Ht);
  }
  return s;
}

// The map of every segment, of the forward pass or (BWD) of what is handed back, which runs against
// it: the lanes' maps of a tile composed by the scan's total, the tiles' one after the other.
template <typename T, bool REV, bool BWD>
__global__ __launch_bounds__(256) void gated_maps_kernel(const Args p) {
  constexpr int V = kV;
  const uint32_t id = group_id<64>();
  const uint32_t row = id / (uint32_t)p.segs;
  if (row >= p.rows) return;
  constexpr bool DOWN = REV != BWD;  // the pass runs from the last tile to the first
  const int lane = threadIdx.x & 63, seg = id % (uint32_t)p.segs;
  const Row<T> r(p, row);
  const int end = max(r.len, 16 / (int)sizeof(T));
  const T* other = !BWD ? r.x : p.gh ? (const T*)p.gh + (long long)row * p.T : r.x;
  const int i0 = seg * p.span, i1 = min(i0 + p.span, p.tiles);
  int t = (DOWN ? p.tiles - 1 - i0 : i0) * kTile + lane * V;
  struct Tile {
    Raw<T, kV, false> x, g;
  } u, v;
  u.x.load(other, t, end);
  u.g.load(r.g, t, end);
  float As = 1.f, Hs = 0.f;
  int i = i0;
  auto step = [&](Tile& tile, Tile& next) __attribute__((always_inline)) {
    float b[V], g[V], a[V], c[V];
    const int now = t;
    t += DOWN ? -kTile : kTile;
    next.x.load(other, t, end);
    next.g.load(r.g, t, end);
    if (now - lane * V >= r.len) return;
    tile.x.settle(now, end);
    tile.g.settle(now, end);
#pragma unroll
    for (int k = 0; k < V; ++k) b[k] = BWD && !p.gh ? 0.f : tile.x[k], g[k] = tile.g[k];
    if (now + V > r.len) hold(r.len - now, g, b);
    float A = 1.f, H = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = DOWN ? V - 1 - q : q;
      gate_of<T>(g[k], a[k], c[k]);
      H = BWD ? a[k] * (b[k] + H) : fmaf(a[k], H, c[k] * b[k]);
      A *= a[k];
    }
    scan<64, DOWN>(A, H, At, Ht);
    Hs = fmaf(At, Hs, Ht);
    As *= At;
  };
  step(u, v);
  while (++i < i1) {
    step(v, u);
    if (++i == i1) break;
    step(u, v);
  }
  if (lane == 0) p.maps[id] = make_float2(As, Hs);
}

// W lanes a row; MULTI: more than one tile (W = 64), in p.segs segments; SHORT: rows shorter than a
// piece (W = 1)
template <typename T, int W, int V, bool REV, bool MULTI, bool SHORT>
__global__ __launch_bounds__(256) void gated_fwd_kernel(const Args p) {
  const uint32_t id = group_id<W>(), row = MULTI ? id / (uint32_t)p.segs : id;
  if (row >= p.rows) return;
  const int seg = MULTI ? id % (uint32_t)p.segs : 0;
  const int i0 = MULTI ? seg * p.span : 0, i1 = MULTI ? min(i0 + p.span, p.tiles) : 1;
  const int lane = threadIdx.x & (W - 1);
  const Row<T> r(p, row);
  const int end = SHORT ? p.T : max(r.len, 16 / (int)sizeof(T));
  T* h = (T*)p.h + (long long)row * p.T;
  float s = p.h0 ? p.h0[row] : 0.f;
  if (MULTI && seg > 0) s = enter(p, row, seg, s);
  int t = (MULTI && REV ? p.tiles - 1 - i0 : i0) * kTile + lane * V;
  struct Tile {
    Raw<T, V, SHORT> x, g;
  } u, v;
  u.x.load(r.x, t, end);
  u.g.load(r.g, t, end);
  int i = i0;
  // one tile; the next one's loads go to registers of their own (copies would wait for them)
  auto step = [&](Tile& tile, Tile& next) __attribute__((always_inline)) {
    if (MULTI && lane == 0) p.carry[(long long)row * p.tiles + (REV ? p.tiles - 1 - i : i)] = s;
    float b[V], g[V], a[V], c[V];
    const int now = t;
    if (MULTI) {
      t += REV ? -kTile : kTile;
      next.x.load(r.x, t, end);
      next.g.load(r.g, t, end);
      if (now - lane * V >= r.len) {  // a tile past the clip's end
        clear(0, b);
        store(h, now, p.T, b);
        return;
      }
    }
    tile.x.settle(now, end);
    tile.g.settle(now, end);
#pragma unroll
    for (int k = 0; k < V; ++k) b[k] = tile.x[k], g[k] = tile.g[k];
    if (now + V > r.len) hold(r.len - now, g, b);
    float A = 1.f, H = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q;
      gate_of<T>(g[k], a[k], c[k]);
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
    if (r.len < p.T && now + V > r.len) clear(r.len - now, b);
    store(h, now, p.T, b);
  };
  step(u, v);
  while (MULTI && ++i < i1) {
    step(v, u);
    if (++i == i1) break;
    step(u, v);
  }
  if ((!MULTI || i1 == p.tiles) && lane == (W == 64 || REV ? 0 : W - 1)) p.last[row] = s;
}

template <typename T, int W, int V, bool REV, bool MULTI, bool SHORT>
__global__ __launch_bounds__(256) void gated_bwd_kernel(const Args p) {
  const uint32_t id = group_id<W>(), row = MULTI ? id / (uint32_t)p.segs : id;
  if (row >= p.rows) return;
  const int seg = MULTI ? id % (uint32_t)p.segs : 0;
  const int i0 = MULTI ? seg * p.span : 0, i1 = MULTI ? min(i0 + p.span, p.tiles) : 1;
  const int lane = threadIdx.x & (W - 1);
  const Row<T> r(p, row);
  const int end = SHORT ? p.T : max(r.len, 16 / (int)sizeof(T));
  const T* gh = p.gh ? (const T*)p.gh + (long long)row * p.T : r.x;
  float s = p.glast ? p.glast[row] : 0.f;
  const float h0 = p.h0 ? p.h0[row] : 0.f;
  if (MULTI && seg > 0) s = enter(p, row, seg, s);
  int t = (MULTI && !REV ? p.tiles - 1 - i0 : i0) * kTile + lane * V;
  struct Tile {
    Raw<T, V, SHORT> x, g, d;
  } v, w;
  v.x.load(r.x, t, end);
  v.g.load(r.g, t, end);
  v.d.load(gh, t, end);
  int i = i0;
  auto step = [&](Tile& tile, Tile& next) __attribute__((always_inline)) {
    const float in = MULTI ? p.carry[(long long)row * p.tiles + (REV ? i : p.tiles - 1 - i)] : h0;
    float x[V], g[V], d[V], a[V], c[V];
    const int now = t;
    if (MULTI) {
      t += REV ? kTile : -kTile;
      next.x.load(r.x, t, end);
      next.g.load(r.g, t, end);
      next.d.load(gh, t, end);
      if (now - lane * V >= r.len) {  // a tile past the clip's end
        clear(0, x);
        store((T*)p.dx + (long long)row * p.T, now, p.T, x);
        store((T*)p.dgate + (long long)row * p.T, now, p.T, x);
        return;
      }
    }
    tile.x.settle(now, end);
    tile.g.settle(now, end);
    tile.d.settle(now, end);
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = tile.x[k], g[k] = tile.g[k], d[k] = p.gh ? tile.d[k] : 0.f;
    if (now + V > r.len) {
      hold(r.len - now, g, x);
      clear(r.len - now, d);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) gate_of<T>(g[k], a[k], c[k]);
    float A = 1.f, H = 0.f, U = 0.f, At, Ht;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int k = REV ? V - 1 - q : q, j = V - 1 - k;
      H = fmaf(a[k], H, c[k] * x[k]);
      A *= a[k];
      U = a[j] * (d[j] + U);
    }
    float Ua = A;
    scan_two<W, REV>(A, H, Ua, U, At, Ht);
    float e = fmaf(A, in, H);  // the state before the lane's first frame
    float u = fmaf(Ua, s, U);  // what the frame after the lane's last hands back
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
    if (r.len < p.T && now + V > r.len) {
      clear(r.len - now, x);
      clear(r.len - now, diff);
    }
    store((T*)p.dx + (long long)row * p.T, now, p.T, x);
    store((T*)p.dgate + (long long)row * p.T, now, p.T, diff);
  };
  step(v, w);
  while (MULTI && ++i < i1) {
    step(w, v);
    if (++i == i1) break;
    step(v, w);
  }
  if (p.dh0 && (!MULTI || i1 == p.tiles) && lane == (W == 64 || !REV ? 0 : W - 1)) p.dh0[row] = s;
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
  gate_of<T>((float)gate[b * gb + c], a, cc);
  const float s = fmaf(a, state[i], cc * (float)x[b * xb + c]);
  state[i] = s;
  h[i] = (T)s;
}

// lanes of a row: the fewest that hold it in one tile
int lanes_of(int32_t T) {
  int w = 1;
  while (w < 64 && w * kV < T) w *= 2;
  return w;
}

int tiles_of(int32_t type, int32_t T) {
  return T <= (type == MST_F32 ? kTile : 64 * kWide) ? 1 : (T + kTile - 1) / kTile;
}

// Tiles of a segment (all of them: one wave a row). A wave takes about 0.8 us a tile forward and 1.1
// us backward whatever the others do, so few rows with a long axis leave the chip idle; segments
// read x and gate (gate and gh) twice and cost a launch. Float32, forward + backward, one wave a row
// -> segments: 128 rows of 50001 frames 76 + 104 -> 27 + 36 us, 512 of 60000 110 + 219 -> 109 + 176, but
// 1024 of 8192 (16 tiles) 20 + 30 -> 31 + 43 and 300 of 3500 (7 tiles) 16 + 17 -> 22 + 23. 8192 waves fill
// the chip's slots (2048 waves: 117 + 197 in the second case). Both bounds lie between those points and are
// not measured close by, nor in 16 bits: few rows of 8 to 19 tiles may be better cut. A segment's last turn
// fetches its neighbour's first tile and drops it (in range, but read for nothing: at two tiles a segment
// the three kernels read 60, 69 and 106 MB where 51, 51 and 77 would do).
int span_of(long long rows, int tiles) {
  if (rows > 640 || tiles < 20) return tiles;
  return (int)((rows * tiles + 8191) / 8192);
}

template <typename T, bool REV, bool BWD>
void launch_w(const Args& p, hipStream_t st) {
  const int w = lanes_of(p.T);
  const dim3 grid((unsigned)(((long long)p.rows * p.segs * w + 255) / 256));
  if (p.segs > 1) hipLaunchKernelGGL((gated_maps_kernel<T, REV, BWD>), grid, dim3(256), 0, st, p);
#define MST_GATED(W_, V_, MULTI, SHORT)                                                                        \
  do {                                                                                                     \
    if (BWD) hipLaunchKernelGGL((gated_bwd_kernel<T, W_, V_, REV, MULTI, SHORT>), grid, dim3(256), 0, st, p);  \
    else hipLaunchKernelGGL((gated_fwd_kernel<T, W_, V_, REV, MULTI, SHORT>), grid, dim3(256), 0, st, p);      \
  } while (0)
  if (p.T < 16 / (int)sizeof(T)) MST_GATED(1, kV, false, true);
  else if (w == 1) MST_GATED(1, kV, false, false);
  else if (w == 2) MST_GATED(2, kV, false, false);
  else if (w == 4) MST_GATED(4, kV, false, false);
  else if (w == 8) MST_GATED(8, kV, false, false);
  else if (w == 16) MST_GATED(16, kV, false, false);
  else if (w == 32) MST_GATED(32, kV, false, false);
  else if (p.T <= kTile) MST_GATED(64, kV, false, false);
  else if (p.tiles > 1) MST_GATED(64, kV, true, false);
  else if constexpr (sizeof(T) == 2) MST_GATED(64, kWide, false, false);
#undef MST_GATED
}

int segs_of(long long rows, int tiles) {
  const int span = span_of(rows, tiles);
  return (tiles + span - 1) / span;
}

// the sizes of a call; false where the workspace is too small
bool set_sizes(Args& p, int32_t type, int32_t B, int32_t C, int32_t T, void* workspace, size_t ws_bytes) {
  p.C = C, p.T = T, p.tiles = tiles_of(type, T), p.rows = (uint32_t)B * (uint32_t)C;
  p.span = span_of(p.rows, p.tiles), p.segs = segs_of(p.rows, p.tiles);
  p.maps = (float2*)workspace;
  return p.segs == 1 || (workspace && ws_bytes >= (size_t)p.rows * p.segs * sizeof(float2));
}

template <bool BWD>
int launch(const Args& p, int type, int reverse, hipStream_t st) {
  if (type == MST_F32) reverse ? launch_w<float, true, BWD>(p, st) : launch_w<float, false, BWD>(p, st);
  else if (type == MST_BF16) reverse ? launch_w<__bf16, true, BWD>(p, st) : launch_w<__bf16, false, BWD>(p, st);
  else reverse ? launch_w<_Float16, true, BWD>(p, st) : launch_w<_Float16, false, BWD>(p, st);
  MST_CHECK_LAUNCH();
  return MST_OK;
}

// (a grid has fewer than 2^32 threads)
bool good_shape(int32_t type, int32_t B, int32_t C, int32_t T) {
  return type >= MST_F32 && type <= MST_F16 && B > 0 && C > 0 && T > 0 && T <= 0x7fffffff - 2 * kTile &&
         (long long)B * C < (1ll << 31) && (long long)B * C * lanes_of(T) < (1ll << 32) - 256;
}

// Whether C values of `z` bytes in each of B rows at `p` lie apart from the B C contiguous values of `wz`
// bytes that are written at `w`, or are these themselves (a thread then reads what it alone writes).
bool apart(const void* p, int64_t stride, int z, const void* w, int wz, int32_t B, int32_t C) {
  if (p == w && z == wz && (B == 1 || stride == C)) return true;
  const __int128 row = (__int128)C * z, s = (uintptr_t)w, e = s + (__int128)B * C * wz;
  __int128 a = (uintptr_t)p, step = (__int128)stride * z;
  if (step < 0) a += step * (B - 1), step = -step;
  if (a >= e || a + step * (B - 1) + row <= s) return true;
  if (a + row <= s) a += ((s - row - a) / step + 1) * step;  // the first row that ends behind the start of w
  return a >= e;
}

}  // namespace

extern "C" {

int32_t mst_gated_tiles(int32_t type, int32_t T) {
  const int tiles = tiles_of(type, T);
  return tiles > 1 ? tiles : 0;
}

size_t mst_gated_workspace_size(int32_t type, int32_t B, int32_t C, int32_t T) {
  if (!good_shape(type, B, C, T)) return 0;
  const long long rows = (long long)B * C;
  const int segs = segs_of(rows, tiles_of(type, T));
  return segs > 1 ? (size_t)rows * segs * sizeof(float2) : 0;
}

int mst_gated_fwd(int32_t type, const void* x, int64_t xb, int64_t xc, const void* gate, int64_t gb,
                  int64_t gc, const float* h0, const int32_t* lengths, int32_t B, int32_t C, int32_t T,
                  int32_t reverse, void* h, float* last, float* carry, void* workspace, size_t ws_bytes,
                  void* stream) {
  MST_REQUIRE(good_shape(type, B, C, T) && x && gate && h && last);
  MST_REQUIRE(tiles_of(type, T) == 1 || carry);
  Args p = {};
  p.x = x, p.xb = xb, p.xc = xc, p.gate = gate, p.gb = gb, p.gc = gc;
  p.h0 = h0, p.len = lengths, p.h = h, p.last = last, p.carry = carry;
  MST_REQUIRE(set_sizes(p, type, B, C, T, workspace, ws_bytes));
  return launch<false>(p, type, reverse, (hipStream_t)stream);
}

int mst_gated_bwd(int32_t type, const void* x, int64_t xb, int64_t xc, const void* gate, int64_t gb,
                  int64_t gc, const float* h0, const int32_t* lengths, const float* carry,
                  const void* gh, const float* glast, int32_t B, int32_t C, int32_t T, int32_t reverse,
                  void* dx, void* dgate, float* dh0, void* workspace, size_t ws_bytes, void* stream) {
  MST_REQUIRE(good_shape(type, B, C, T) && x && gate && dx && dgate);
  MST_REQUIRE(tiles_of(type, T) == 1 || carry);
  Args p = {};
  p.x = x, p.xb = xb, p.xc = xc, p.gate = gate, p.gb = gb, p.gc = gc;
  p.h0 = h0, p.len = lengths, p.carry = const_cast<float*>(carry);
  p.gh = gh, p.glast = glast, p.dx = dx, p.dgate = dgate, p.dh0 = dh0;
  MST_REQUIRE(set_sizes(p, type, B, C, T, workspace, ws_bytes));
  return launch<true>(p, type, reverse, (hipStream_t)stream);
}

int mst_gated_step(int32_t type, const void* x, int64_t xb, const void* gate, int64_t gb, int32_t B,
                   int32_t C, float* state, void* h, void* stream) {
  MST_REQUIRE(good_shape(type, B, C, 1) && x && gate && state && h);
  const int z = type == MST_F32 ? 4 : 2;
  MST_REQUIRE(apart(x, xb, z, state, 4, B, C) && apart(gate, gb, z, state, 4, B, C));
  MST_REQUIRE(apart(x, xb, z, h, z, B, C) && apart(gate, gb, z, h, z, B, C));
  MST_REQUIRE(apart(h, C, z, state, 4, B, C));
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
