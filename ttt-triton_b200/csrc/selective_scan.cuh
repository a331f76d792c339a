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
inline int save_every(int N) { return 32 / shape_of(N).NPT; }


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

// Stages rows t0 .. t0 + TT - 1 of B or C as fp32 in shared memory (0 past the end, past N and
// for tokens of no sequence). `quads`: four states at a time, where every row is N = NP states
// on a boundary of four.
template <typename T, int NP, int TT, int THREADS>
__device__ __forceinline__ void stage_rows(float* dst, const T* src, long long ld, int t0, int t1, int N,
                                           const int* seq, bool quads) {
  if (quads) {
    struct alignas(4 * sizeof(T)) Quad {
      T v[4];
    };
#pragma unroll
    for (int k = 0; k < (TT * NP / 4 + THREADS - 1) / THREADS; ++k) {
      const int i = threadIdx.x + k * THREADS, t = i / (NP / 4), n = i % (NP / 4) * 4;
      if (TT * NP / 4 % THREADS == 0 || i < TT * NP / 4) {
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (t0 + t < t1 && !(seq && seq[t0 + t] < 0)) {
          const Quad q = *reinterpret_cast<const Quad*>(src + (t0 + t) * ld + n);
          f = make_float4(to_f(q.v[0]), to_f(q.v[1]), to_f(q.v[2]), to_f(q.v[3]));
        }
        *reinterpret_cast<float4*>(dst + i * 4) = f;
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < TT * NP; i += THREADS) {
    const int t = i / NP, n = i - t * NP;
    dst[i] = t0 + t < t1 && n < N && !(seq && seq[t0 + t] < 0) ? to_f(src[(t0 + t) * ld + n]) : 0.f;
  }
}

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
// max |x| that keeps a NaN (as integer bits it is above all numbers)
__device__ __forceinline__ unsigned max_bits(unsigned m, float2 x) {
  return max(m, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
}

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

// The sums over the LN threads of two adjacent channels.
template <int LN>
__device__ __forceinline__ float2 state_sums(const float* y) {
  if constexpr (LN == 1) return *reinterpret_cast<const float2*>(y);
  if constexpr (LN == 2) {
    const float4 v = *reinterpret_cast<const float4*>(y);
    return make_float2(v.x + v.y, v.z + v.w);
  }
  float2 r = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < LN / 4; ++j) {
    const float4 v = reinterpret_cast<const float4*>(y)[j], x = reinterpret_cast<const float4*>(y + LN)[j];
    r = __fadd2_rn(r, make_float2((v.x + v.y) + (v.z + v.w), (x.x + x.y) + (x.z + x.w)));
  }
  return r;
}

// 2^x for the products x = dt A2 of a pair of states. The special-function unit gives 16 an SM
// and clock, the fused multiply-add pipes stand half idle beside it, so a part of the pairs
// goes there: x = k + f, 2^f = 1 + f q(f) with q of degree 4 (relative error 1.2e-7, and that
// of a rounding near 1, where decays act longest), k into the exponent. That form holds for
// |x| < 126 only; kernels look at a tile's largest |dt| times the largest |A2| first.
constexpr float kPolyRange = 126.f;
__device__ __forceinline__ float2 pow2_poly(float2 dt, float2 A2) {
  const float2 magic = make_float2(12582912.f, 12582912.f);  // 1.5 * 2^23: the sum's low bits are k
  const float2 xi = __ffma2_rn(dt, A2, magic);
  const float2 k = __fadd2_rn(xi, make_float2(-12582912.f, -12582912.f));
  const float2 f = __ffma2_rn(dt, A2, make_float2(-k.x, -k.y));
  float2 q = __ffma2_rn(f, make_float2(0.0013405575882643461f, 0.0013405575882643461f),
                        make_float2(0.009670727886259556f, 0.009670727886259556f));
  q = __ffma2_rn(f, q, make_float2(0.05550314858555794f, 0.05550314858555794f));
  q = __ffma2_rn(f, q, make_float2(0.24022258818149567f, 0.24022258818149567f));
  q = __ffma2_rn(f, q, make_float2(0.6931471824645996f, 0.6931471824645996f));
  q = __ffma2_rn(f, q, make_float2(1.f, 1.f));
  return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(xi.x) << 23)),
                     __int_as_float(__float_as_int(q.y) + (__float_as_int(xi.y) << 23)));
}
__device__ __forceinline__ float2 pow2_unit(float2 dt, float2 A2) {
  const float2 x = __fmul2_rn(dt, A2);
  return make_float2(ex2(x.x), ex2(x.y));
}

// The largest |x| of a CTA as integer bits: per warp, for a tile's readers.
template <int WARPS>
__device__ __forceinline__ float max_of(const unsigned (&m)[WARPS]) {
  unsigned v = m[0];
#pragma unroll
  for (int k = 1; k < WARPS; ++k) v = max(v, m[k]);
  return __uint_as_float(v);
}

// Start, end and membership of the tile's tokens as bit masks (at most 32 tokens).
struct SeqMask {
  unsigned start, end, in;
};
__device__ __forceinline__ bool in_sequence(const int* seq, int t) { return !seq || seq[t] >= 0; }
template <int TT>
__device__ __forceinline__ void stage_masks(SeqMask* m, const int* seq, int t0, int t1, int T) {
  if (threadIdx.x < 32) {
    const int t = t0 + threadIdx.x;
    const bool on = threadIdx.x < TT && t < t1;
    const unsigned s = __ballot_sync(0xffffffffu, on && seq_starts(seq, t));
    const unsigned e = __ballot_sync(0xffffffffu, on && seq_ends(seq, t, T));
    const unsigned v = __ballot_sync(0xffffffffu, on && seq[t] >= 0);
    if (threadIdx.x == 0) m->start = s, m->end = e, m->in = v;
  }
}

// Launches the pass over pieces (local end states, then the states entering each piece), when
// the time axis is split. REV: the backward recurrence's carries instead of the states.
int chunk_states(const Params& p, int dt, bool rev, cudaStream_t st, const char* who);
// Splits the time axis and lays its part of the scratch out behind `extra` bytes of the caller.
int plan(Params& p, void* scratch, size_t scratch_bytes, size_t extra, const char* who);
bool quads(const Params& p, int dt);
bool couples(const Params& p, int dt);
size_t plan_bytes(int rows, int L, int D, int N);
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
