// Parameters, sizes and the split of the selective scan, shared by its forward, backward and
// single-token kernels.
//
//   dt = softplus(delta + bias);  h[t] = exp(dt A) h[t-1] + dt u B[t];  y = <h, C[t]> + D u;
//   out = y z sigmoid(z)
//
// per channel d with N states; B and C are shared by the D / G channels of a group.
#pragma once

#include "scan_common.cuh"

namespace ttt {
namespace scan {

constexpr int kMaxStates = 128;

struct Params {
  int rows, L, D, G, N;
  int Dg;        // channels of a group
  int tiles;     // channel tiles of a group
  int nchunks;   // pieces of the time axis
  int chunk;     // tokens of a piece
  int nsave;     // saved states of a row
  const void *u, *delta, *B, *C, *z;
  long long u_b, u_l, delta_b, delta_l, B_b, B_l, B_g, C_b, C_l, C_g, z_b, z_l;  // element strides
  const float *A, *Dskip, *bias;
  int softplus;
  int quads;           // rows of B and C are read four states at a time
  int couples;         // activations are read and written two channels at a time
  const int* seq;      // packed rows: each token's sequence (rows == 1), else NULL
  const float* init;   // [sequences, D, N] or NULL
  float* fin;          // [sequences, D, N] or NULL
  void* out;           // [rows, L, D]
  float* hsave;        // [rows, nsave, D, N]: the state before every save_every()-th token, or NULL
  float* cstate;       // [rows, nchunks, D, N]: the state entering each piece (nchunks > 1)
  float* csum;         // [rows, nchunks, D]: the sum of dt over a piece
  // backward
  const void* dout;    // [rows, L, D]
  const float* dfin;   // [sequences, D, N] or NULL
  void *du, *ddelta, *dz;
  float* dinit;        // [sequences, D, N] or NULL
  float *part_B, *part_C;  // [tiles, rows * L, G, N]
  float* part_p;           // [rows * nchunks, D * (N + 2)]: dA | dD | dbias
};

// States per thread and threads per channel for N states. A channel's states lie on the LN
// threads in runs of NPT.
struct Shape {
  int LN, NPT;
};
inline Shape shape_of(int N) {
  if (N <= 4) return {1, 4};
  if (N <= 8) return {2, 4};
  if (N <= 16) return {4, 4};
  if (N <= 32) return {8, 4};
  if (N <= 64) return {8, 8};
  return {8, 16};
}
// Tokens between two saved states: those whose states the backward kernel holds in registers.
__host__ __device__ constexpr int save_every_of(int NPT) { return NPT == 16 ? 2 : 4; }
inline int save_every(int N) { return save_every_of(shape_of(N).NPT); }

// This thread's NPT states of channel d of a [.., D, N] array (0 past N); in fours where N is a
// multiple of four and the array lies on a 16-byte boundary, as torch's allocations do.
template <int NPT>
__device__ __forceinline__ void load_states(const float* base, int d, int n0, int N, bool on, float (&h)[NPT]) {
  const float* p = base + (long long)d * N + n0;
  if (N % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < NPT; i += 4) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (on && n0 + i < N) q = *reinterpret_cast<const float4*>(p + i);
      h[i] = q.x, h[i + 1] = q.y, h[i + 2] = q.z, h[i + 3] = q.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NPT; ++i) h[i] = on && n0 + i < N ? p[i] : 0.f;
}
template <int NPT>
__device__ __forceinline__ void store_states(float* base, int d, int n0, int N, bool on, const float (&h)[NPT]) {
  float* p = base + (long long)d * N + n0;
  if (N % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < NPT; i += 4)
      if (on && n0 + i < N) *reinterpret_cast<float4*>(p + i) = make_float4(h[i], h[i + 1], h[i + 2], h[i + 3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < NPT; ++i)
    if (on && n0 + i < N) p[i] = h[i];
}

// Rows t0 .. t0 + TT - 1 of B or C on their way to shared memory as fp32 (0 past the end, past
// N and for tokens of no sequence): fetch() has four states at a time in registers, where
// every row is N = NP states on a boundary of four (`quads`); put() writes them, or reads and
// writes state by state.
template <typename T, int NP, int TT, int THREADS>
struct Rows {
  static constexpr int Q = (TT * NP / 4 + THREADS - 1) / THREADS;
  struct alignas(4 * sizeof(T)) Quad {
    T v[4];
  };
  Quad q[Q];
  __device__ __forceinline__ void fetch(int tid, const T* src, long long ld, int t0, int t1, const int* seq, bool quads) {
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int i = tid + k * THREADS, t = i / (NP / 4), n = i % (NP / 4) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) q[k].v[e] = from_f<T>(0.f);
      if (quads && (TT * NP / 4 % THREADS == 0 || i < TT * NP / 4) && t0 + t < t1 && !(seq && seq[t0 + t] < 0))
        q[k] = *reinterpret_cast<const Quad*>(src + (t0 + t) * ld + n);
    }
  }
  __device__ __forceinline__ void put(int tid, float* dst, const T* src, long long ld, int t0, int t1, int N, const int* seq,
                                      bool quads) const {
    if (quads) {
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const int i = tid + k * THREADS;
        if (TT * NP / 4 % THREADS == 0 || i < TT * NP / 4)
          *reinterpret_cast<float4*>(dst + i * 4) =
              make_float4(to_f(q[k].v[0]), to_f(q[k].v[1]), to_f(q[k].v[2]), to_f(q[k].v[3]));
      }
      return;
    }
    for (int i = tid; i < TT * NP; i += THREADS) {
      const int t = i / NP, n = i - t * NP;
      dst[i] = t0 + t < t1 && n < N && !(seq && seq[t0 + t] < 0) ? to_f(src[(t0 + t) * ld + n]) : 0.f;
    }
  }
};
// Two adjacent channels of an activation. `both`: one access for the two, where every row has
// them on a boundary of two; else each by itself, where it is there.
template <typename T>
struct Two {  // 16-bit types: one register
  unsigned v;
};
template <>
struct Two<float> {
  float2 v;
};
template <typename T>
__device__ __forceinline__ Two<T> load_two(const T* p, bool on0, bool on1, bool both) {
  Two<T> r;
  if constexpr (std::is_same<T, float>::value) {
    r.v = make_float2(0.f, 0.f);
    if (both) {
      if (on0) r.v = *reinterpret_cast<const float2*>(p);
    } else {
      if (on0) r.v.x = p[0];
      if (on1) r.v.y = p[1];
    }
  } else {
    r.v = 0;
    if (both) {
      if (on0) r.v = *reinterpret_cast<const unsigned*>(p);
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
      if (on0) r.v = q[0];
      if (on1) r.v |= (unsigned)q[1] << 16;
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float2 two_f(const Two<T>& r) {
  if constexpr (std::is_same<T, float>::value) {
    return r.v;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(r.v << 16), __uint_as_float(r.v & 0xffff0000u));
  } else {
    __half2 h;
    memcpy(&h, &r.v, 4);
    return __half22float2(h);
  }
}
template <typename T>
__device__ __forceinline__ void store_two(T* p, float2 v, bool on0, bool on1, bool both) {
  if constexpr (std::is_same<T, float>::value) {
    if (both) {
      if (on0) *reinterpret_cast<float2*>(p) = v;
    } else {
      if (on0) p[0] = v.x;
      if (on1) p[1] = v.y;
    }
  } else {
    unsigned r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 h = __float22bfloat162_rn(v);
      memcpy(&r, &h, 4);
    } else {
      const __half2 h = __float22half2_rn(v);
      memcpy(&r, &h, 4);
    }
    if (both) {
      if (on0) *reinterpret_cast<unsigned*>(p) = r;
    } else {
      unsigned short* q = reinterpret_cast<unsigned short*>(p);
      if (on0) q[0] = (unsigned short)r;
      if (on1) q[1] = (unsigned short)(r >> 16);
    }
  }
}
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }
__device__ __forceinline__ float2 all2(float x) { return make_float2(x, x); }
// sigmoid and softplus (scan_common.cuh) of two
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  const float2 m = __fmul2_rn(x, all2(-kLog2e));
  const float2 e = __fadd2_rn(make_float2(ex2(m.x), ex2(m.y)), all2(1.f));
  return make_float2(rcp(e.x), rcp(e.y));
}
__device__ __forceinline__ float2 softplus2(float2 x) {
  const float2 m = __fmul2_rn(make_float2(fabsf(x.x), fabsf(x.y)), all2(-kLog2e));
  const float2 w = make_float2(ex2(m.x), ex2(m.y)), e = __fadd2_rn(w, all2(2.f));
  const float2 s = __fmul2_rn(w, make_float2(rcp(e.x), rcp(e.y))), v = __fmul2_rn(s, s);
  float2 q = __ffma2_rn(v, all2(0.2814132571220398f), all2(0.2797023057937622f));
  q = __ffma2_rn(v, q, all2(0.4002406597137451f));
  q = __ffma2_rn(v, q, all2(0.666663408279419f));
  q = __ffma2_rn(v, q, all2(2.f));
  return __ffma2_rn(s, q, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}
// x sigmoid(x)
__device__ __forceinline__ float2 silu2(float2 x) { return __fmul2_rn(x, sigmoid2(x)); }
// NPT states as pairs, and a tile row's values for them.
template <int NPT>
struct Pairs {
  float2 v[NPT / 2];
};
template <int NPT>
__device__ __forceinline__ Pairs<NPT> pairs_of(const float (&x)[NPT]) {
  Pairs<NPT> r;
#pragma unroll
  for (int j = 0; j < NPT / 2; ++j) r.v[j] = make_float2(x[2 * j], x[2 * j + 1]);
  return r;
}
template <int NPT>
__device__ __forceinline__ void unpair(const Pairs<NPT>& x, float (&y)[NPT]) {
#pragma unroll
  for (int j = 0; j < NPT / 2; ++j) y[2 * j] = x.v[j].x, y[2 * j + 1] = x.v[j].y;
}
// The states of a thread's two channels, d and d + 1.
template <int NPT>
struct Both {
  Pairs<NPT> c[2];
};
template <int NPT>
__device__ __forceinline__ Both<NPT> load_both(const float* base, int d, int n0, int N, bool on0, bool on1) {
  Both<NPT> r;
  float x[NPT];
  load_states<NPT>(base, d, n0, N, on0, x);
  r.c[0] = pairs_of<NPT>(x);
  load_states<NPT>(base, d + 1, n0, N, on1, x);
  r.c[1] = pairs_of<NPT>(x);
  return r;
}
template <int NPT>
__device__ __forceinline__ void store_both(float* base, int d, int n0, int N, bool on0, bool on1, const Both<NPT>& h) {
  float x[NPT];
  unpair(h.c[0], x);
  store_states<NPT>(base, d, n0, N, on0, x);
  unpair(h.c[1], x);
  store_states<NPT>(base, d + 1, n0, N, on1, x);
}
template <int NPT>
__device__ __forceinline__ Pairs<NPT> row_pairs(const float* row) {  // 16-byte aligned
  Pairs<NPT> r;
#pragma unroll
  for (int j = 0; j < NPT / 4; ++j) {
    const float4 q = reinterpret_cast<const float4*>(row)[j];
    r.v[2 * j] = make_float2(q.x, q.y), r.v[2 * j + 1] = make_float2(q.z, q.w);
  }
  return r;
}

__device__ __forceinline__ float2 params_of(const float* v, int d, bool on0, bool on1) {
  return make_float2(v && on0 ? v[d] : 0.f, v && on1 ? v[d + 1] : 0.f);
}

// exp(dt A) of a pair of states, A2 = A log2(e). The unit's 2^x cuts its argument off: for
// arguments of -0.5 to -0.001 its results were 0.3 * 2^-24 too small on average, which a state
// that is kept for a thousand tokens multiplies. Half a step of 2^-24 on the argument brings
// the average to 0.05 * 2^-24 and costs nothing (a fused multiply-add for a product); a step
// size of zero still gives exactly 1.
constexpr float kHalfStep = 2.9802322387695312e-8f;  // 2^-25
__device__ __forceinline__ float2 decay(float2 dt, float2 A2) {
  const float2 x = __ffma2_rn(dt, A2, all2(kHalfStep));
  return make_float2(ex2(x.x), ex2(x.y));
}

// Start, end and membership of the tile's tokens as bit masks (at most 32 tokens).
struct SeqMask {
  unsigned start, end, in;
};
template <int TT>
__device__ __forceinline__ SeqMask warp_masks(const int* seq, int t0, int t1, int T) {
  const int t = t0 + (threadIdx.x & 31);
  const bool on = (threadIdx.x & 31) < TT && t < t1;
  SeqMask m;
  m.start = __ballot_sync(0xffffffffu, on && seq_starts(seq, t));
  m.end = __ballot_sync(0xffffffffu, on && seq_ends(seq, t, T));
  m.in = __ballot_sync(0xffffffffu, on && seq[t] >= 0);
  return m;
}
__device__ __forceinline__ bool in_sequence(const int* seq, int t) { return !seq || seq[t] >= 0; }
// Launches the pass over pieces (local end states, then the states entering each piece), when
// the time axis is split. REV: the backward recurrence's carries instead of the states.
int chunk_states(const Params& p, int dt, bool rev, cudaStream_t st, const char* who);
// How the time axis is split, the scratch that takes (bytes), and its place behind `extra`
// bytes of the caller's.
void plan_pieces(Params& p, bool backward);
size_t piece_bytes(const Params& p);
int plan_scratch(Params& p, void* scratch, size_t scratch_bytes, size_t extra, const char* who);
bool quads(const Params& p, int dt);
bool couples(const Params& p, int dt);
int check_sizes(const char* who, int rows, int L, int D, int G, int N, int dt);

template <typename F>
int dispatch(int N, F&& f) {
  using std::integral_constant;
  const Shape s = shape_of(N);
  if (s.LN == 1) return f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  if (s.LN == 2) return f(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  if (s.LN == 4) return f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  if (s.NPT == 4) return f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  if (s.NPT == 8) return f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  return f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
}

// Block -> (row, piece, group, first channel of the tile within the group)
struct Where {
  int row, piece, g, d0;
};
template <int DT>
__device__ __forceinline__ Where where(const Params& p) {
  long long i = blockIdx.x;
  const int tile = i % (p.tiles * p.G);
  i /= p.tiles * p.G;
  Where w;
  w.piece = i % p.nchunks;
  w.row = i / p.nchunks;
  w.g = tile / p.tiles;
  w.d0 = (tile - w.g * p.tiles) * DT;
  return w;
}

}  // namespace scan
}  // namespace ttt
