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
  const int* seq;      // packed rows: each token's sequence (rows == 1), else NULL
  const float* init;   // [sequences, D, N] or NULL
  float* fin;          // [sequences, D, N] or NULL
  void* out;           // [rows, L, D]
  float* hsave;        // [rows, nsave, D, N]: the state before every TB-th token, or NULL
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
// Tokens between two saved states: the backward kernel's time tile.
inline int save_every(int N) { return 64 / shape_of(N).NPT; }

__device__ __forceinline__ float step_size(const Params& p, float raw) { return p.softplus ? softplus(raw) : raw; }

// Loads this thread's NPT states of channel d from a [.., D, N] array (0 past N).
template <int NPT>
__device__ __forceinline__ void load_states(const float* base, int d, int n0, int N, bool on, float (&h)[NPT]) {
#pragma unroll
  for (int i = 0; i < NPT; ++i) h[i] = on && n0 + i < N ? base[(long long)d * N + n0 + i] : 0.f;
}
template <int NPT>
__device__ __forceinline__ void store_states(float* base, int d, int n0, int N, bool on, const float (&h)[NPT]) {
#pragma unroll
  for (int i = 0; i < NPT; ++i)
    if (on && n0 + i < N) base[(long long)d * N + n0 + i] = h[i];
}

// Stages rows t0 .. t0 + TT - 1 of B or C as fp32 in shared memory (0 past the end, past N and
// for tokens of no sequence).
template <typename T, int NP, int TT, int THREADS>
__device__ __forceinline__ void stage_rows(float* dst, const T* src, long long ld, int t0, int t1, int N,
                                           const int* seq) {
  for (int i = threadIdx.x; i < TT * NP; i += THREADS) {
    const int t = i / NP, n = i - t * NP;
    dst[i] = t0 + t < t1 && n < N && !(seq && seq[t0 + t] < 0) ? to_f(src[(t0 + t) * ld + n]) : 0.f;
  }
}

// Start, end and membership of the tile's tokens as bit masks (at most 32 tokens).
struct SeqMask {
  unsigned start, end, in;
};
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
