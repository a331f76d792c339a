// Selective state space scan, forward: prompts, packed prompts and the training forward, and
// the single-token step. The recurrence is in selective_scan.cuh.
//
// A channel's N states are split over LN threads, NPT in each and two channels a thread, and
// stay in registers while the CTA walks the time axis tile by tile: a tile's step sizes and
// inputs are worked out once per (token, channel) into shared memory, then every thread runs
// its states through the tile's tokens, then the partial outputs of a channel's threads are
// added, the skip and the gate applied and the result written. One exponential per (token,
// channel, state) is its floor; the unit is half busy, and the fixed latency of the recurrence's
// instructions at 24 warps an SM bounds it (16 x 2048 x 1536, 16 states: 408 us, floor 179).
// Shared-memory reads cost bytes per thread whether or not threads read the same: the second
// channel halves those of B and C.
//
// With few channels in all, the time axis is split into pieces: a first pass finds each
// piece's end state from zero and the sum of its step sizes (its whole decay is
// exp(A * sum)), a second runs over the pieces, and the main pass starts each piece from
// the state that enters it.
#include "selective_scan.cuh"

namespace ttt {
namespace scan {

template <int LN, int NPT>
struct Fwd {
  static constexpr int HALF = 128;                   // threads of the recurrence; as many for the element-wise work
  static constexpr int THREADS = 2 * HALF;
  static constexpr int DT = 2 * HALF / LN;           // channels of a CTA
  static constexpr int NP = LN * NPT;                // states, padded
  static constexpr int TT = LN >= 4 ? 16 : 8;      // tokens of a tile
  static constexpr int RUN = 8;                      // tokens unrolled
  static constexpr int TWOS = TT / LN;               // couples of channels of a thread, one token each
  static constexpr int STEP = LN;                    // tokens between them
  static constexpr int YS = DT + (LN > 1 ? 32 / LN : 0);  // row of partial outputs, padded off bank conflicts
  struct Tile {
    float B[TT * NP], C[TT * NP];
    float2 d[TT * DT];       // step size, step size * input
    float y[TT * LN * YS];   // partial outputs
  };
  struct Smem {
    Tile tile[2];
  };
};

// A thread of the recurrence: states n0 .. of channels d, d + 1.
template <int LN, int NPT>
struct Lane {
  int nl, n0, cl, d;
  bool c0, c1;
  __device__ __forceinline__ Lane(const Params& p, const Where& w) {
    const int tid = threadIdx.x;
    nl = tid % LN, n0 = nl * NPT, cl = tid / LN * 2;
    d = w.g * p.Dg + w.d0 + cl;
    c0 = w.d0 + cl < p.Dg, c1 = w.d0 + cl + 1 < p.Dg;
  }
};
// A thread of the element-wise work: channels pd, pd + 1 at tokens tq, tq + STEP, .. of a tile.
template <int LN, int NPT>
struct Couple {
  int tid, pc, tq, pd;
  bool on0, on1;
  __device__ __forceinline__ Couple(const Params& p, const Where& w) {
    using F = Fwd<LN, NPT>;
    tid = threadIdx.x - F::HALF;
    pc = tid % (F::DT / 2) * 2, tq = tid / (F::DT / 2);
    pd = w.g * p.Dg + w.d0 + pc;
    on0 = w.d0 + pc < p.Dg, on1 = w.d0 + pc + 1 < p.Dg;
  }
};

template <int LN, int NPT>
__device__ __forceinline__ Both<NPT> load_both(const float* base, const Lane<LN, NPT>& q, int N, bool on) {
  return load_both<NPT>(base, q.d, q.n0, N, on && q.c0, on && q.c1);
}
template <int LN, int NPT>
__device__ __forceinline__ void store_both(float* base, const Lane<LN, NPT>& q, int N, bool on, const Both<NPT>& h) {
  store_both<NPT>(base, q.d, q.n0, N, on && q.c0, on && q.c1, h);
}
// A2 = A log2(e)
template <int LN, int NPT>
__device__ __forceinline__ Both<NPT> load_decays(const Params& p, const Lane<LN, NPT>& q) {
  Both<NPT> A2 = load_both(p.A, q, p.N, true);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < NPT / 2; ++j) A2.c[c].v[j] = __fmul2_rn(A2.c[c].v[j], all2(kLog2e));
  return A2;
}

// The CTA's barrier for its two halves, which wait at places of their own in the code.
__device__ __forceinline__ void tile_barrier() { asm volatile("barrier.sync 1, 256;" ::: "memory"); }

// The recurrence over one tile, by the first half of the CTA. STATE: states only, no outputs;
// REV: backwards, h = a (h + x R).
template <int LN, int NPT, bool SEQ, bool STATE, bool REV>
__device__ __forceinline__ void run_tile(const Params& p, const Where& w, const Lane<LN, NPT>& q,
                                         typename Fwd<LN, NPT>::Tile& s, const Both<NPT>& A2, Both<NPT>& h,
                                         int t0, int tend, const float* edge) {
  using F = Fwd<LN, NPT>;
  const long long DN = (long long)p.D * p.N;
  constexpr int every = save_every_of(NPT);
  SeqMask mask{};
  if (SEQ) mask = warp_masks<F::TT>(p.seq, t0, tend, p.L);
  const unsigned edges = REV ? mask.end : STATE ? mask.start : mask.start | mask.end;
#pragma unroll 1
  for (int r0 = 0; r0 < F::TT; r0 += F::RUN) {
    const int r = REV ? F::TT - F::RUN - r0 : r0;
    if (t0 + r >= tend) continue;
    const auto tokens = [&](auto checks) {
#pragma unroll
      for (int k = 0; k < F::RUN; ++k) {
        const int t = r + (REV ? F::RUN - 1 - k : k);
        if constexpr (decltype(checks)::value) {
          if (t0 + t >= tend) continue;
        }
        if (!STATE && k % every == 0 && p.hsave)
          store_both(p.hsave + ((long long)w.row * p.nsave + (t0 + t) / every) * DN, q, p.N, true, h);
        if constexpr (decltype(checks)::value && SEQ) {
          if ((REV ? mask.end : mask.start) >> t & 1) {
            const int sq = p.seq[t0 + t];
            h = load_both(edge + sq * DN, q, p.N, sq >= 0 && edge);
          }
        }
        const float4 d4 = *reinterpret_cast<const float4*>(&s.d[t * F::DT + q.cl]);
        const Pairs<NPT> B2 = row_pairs<NPT>(s.B + t * F::NP + q.n0);
        Pairs<NPT> C2;
        if (!STATE) C2 = row_pairs<NPT>(s.C + t * F::NP + q.n0);
        float2 y = all2(0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 dt = all2(c ? d4.z : d4.x), x = all2(c ? d4.w : d4.y);
          float2 sum = all2(0.f);
#pragma unroll
          for (int j = 0; j < NPT / 2; ++j) {
            const float2 a = decay(dt, A2.c[c].v[j]);
            float2& hj = h.c[c].v[j];
            if constexpr (REV) hj = __fmul2_rn(a, __ffma2_rn(x, B2.v[j], hj));
            else hj = __ffma2_rn(a, hj, __fmul2_rn(x, B2.v[j]));
            if (!STATE) sum = j ? __ffma2_rn(hj, C2.v[j], sum) : __fmul2_rn(hj, C2.v[j]);
          }
          (c ? y.y : y.x) = sum.x + sum.y;
        }
        if (!STATE) *reinterpret_cast<float2*>(&s.y[(t * LN + q.nl) * F::YS + q.cl]) = y;
        if constexpr (decltype(checks)::value && SEQ && !STATE) {
          if (p.fin && (mask.end >> t & 1)) {
            const int sq = p.seq[t0 + t];
            store_both(p.fin + sq * DN, q, p.N, sq >= 0, h);
          }
        }
      }
    };
    if (t0 + r + F::RUN > tend || (SEQ && (edges >> r & 0xff))) tokens(std::true_type{});
    else tokens(std::false_type{});
  }
}

// The first half of the CTA runs tile i while the second finishes the outputs of tile i - 1 and
// prepares tile i + 1 in the other buffer; one barrier a tile.
template <typename T, int LN, int NPT, bool SEQ>
__global__ void __launch_bounds__(256, NPT == 4 ? 3 : NPT == 8 ? 2 : 1) scan_fwd_kernel(const __grid_constant__ Params p) {
  using F = Fwd<LN, NPT>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const int ntiles = (tend - tbeg + F::TT - 1) / F::TT;
  const long long DN = (long long)p.D * p.N;

  if (threadIdx.x < F::HALF) {
    const Lane<LN, NPT> q(p, w);
    const Both<NPT> A2 = load_decays(p, q);
    Both<NPT> h = p.nchunks > 1 ? load_both(p.cstate + ((long long)w.row * p.nchunks + w.piece) * DN, q, p.N, true)
                                : load_both(p.init + w.row * DN, q, p.N, p.init && !SEQ);
    for (int i = 0; i < ntiles; ++i) {
      tile_barrier();
      run_tile<LN, NPT, SEQ, false, false>(p, w, q, s.tile[i & 1], A2, h, tbeg + i * F::TT, tend, p.init);
    }
    tile_barrier();
    if (!SEQ && p.fin && tend == p.L) store_both(p.fin + w.row * DN, q, p.N, true, h);
    return;
  }

  const Couple<LN, NPT> q(p, w);
  const int* seq = SEQ ? p.seq : nullptr;
  const float2 skip = params_of(p.Dskip, q.pd, q.on0, q.on1), bias = params_of(p.bias, q.pd, q.on0, q.on1);
  const T* u = static_cast<const T*>(p.u) + w.row * p.u_b + q.pd;
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + q.pd;
  const T* z = static_cast<const T*>(p.z) + w.row * p.z_b + q.pd;
  const T* B = static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const T* C = static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g;
  T* out = static_cast<T*>(p.out) + (long long)w.row * p.L * p.D + q.pd;
  // inputs and gates of the tile that is prepared, the one that runs and the one before
  Two<T> u2[F::TWOS], z2[F::TWOS], u1[F::TWOS], z1[F::TWOS], u0[F::TWOS], z0[F::TWOS], dd[F::TWOS];
  Rows<T, F::NP, F::TT, F::HALF> rB, rC;
  for (int i = -1; i <= ntiles; ++i) {
    const int tn = tbeg + (i + 1) * F::TT, tl = tbeg + (i - 1) * F::TT;
    if (i + 1 < ntiles) {
#pragma unroll
      for (int k = 0; k < F::TWOS; ++k) {
        const int tok = tn + q.tq + k * F::STEP;
        const bool in = tok < tend && in_sequence(seq, tok), on0 = in && q.on0, on1 = in && q.on1;
        dd[k] = load_two(delta + tok * p.delta_l, on0, on1, p.couples), u2[k] = load_two(u + tok * p.u_l, on0, on1, p.couples);
        z2[k] = load_two(z + tok * p.z_l, on0 && p.z, on1 && p.z, p.couples);
      }
      rB.fetch(q.tid, B, p.B_l, tn, tend, seq, p.quads), rC.fetch(q.tid, C, p.C_l, tn, tend, seq, p.quads);
    }
    if (i >= 1) {
      const auto& tile = s.tile[(i - 1) & 1];
#pragma unroll
      for (int k = 0; k < F::TWOS; ++k) {
        const int t = q.tq + k * F::STEP, tok = tl + t;
        float2 y = __fmul2_rn(skip, two_f(u0[k]));
#pragma unroll
        for (int j = 0; j < LN; ++j)
          y = __fadd2_rn(y, *reinterpret_cast<const float2*>(&tile.y[(t * LN + j) * F::YS + q.pc]));
        if (p.z) y = __fmul2_rn(y, silu2(two_f(z0[k])));
        if (SEQ && tok < tend && seq[tok] < 0) y = all2(0.f);  // a token of no sequence
        store_two(out + (long long)tok * p.D, y, q.on0 && tok < tend, q.on1 && tok < tend, p.couples);
      }
    }
    if (i + 1 < ntiles) {
      auto& tile = s.tile[(i + 1) & 1];
#pragma unroll
      for (int k = 0; k < F::TWOS; ++k) {
        const int t = q.tq + k * F::STEP, tok = tn + t;
        float2 dt = __fadd2_rn(two_f(dd[k]), bias);
        if (p.softplus) dt = softplus2(dt);
        if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
        const float2 x = __fmul2_rn(dt, two_f(u2[k]));
        *reinterpret_cast<float4*>(&tile.d[t * F::DT + q.pc]) = make_float4(dt.x, x.x, dt.y, x.y);
      }
      rB.put(q.tid, tile.B, B, p.B_l, tn, tend, p.N, seq, p.quads);
      rC.put(q.tid, tile.C, C, p.C_l, tn, tend, p.N, seq, p.quads);
    }
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) u0[k] = u1[k], z0[k] = z1[k], u1[k] = u2[k], z1[k] = z2[k];
    if (i < ntiles) tile_barrier();
  }
}

// A piece's end state from zero (REV: the carry that leaves its first token from zero at its
// last), and the sum of its step sizes.
template <typename T, int LN, int NPT, bool REV, bool SEQ>
__global__ void __launch_bounds__(256, NPT == 4 ? 3 : NPT == 8 ? 2 : 1) scan_chunk_kernel(const __grid_constant__ Params p) {
  using F = Fwd<LN, NPT>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const int ntiles = (tend - tbeg + F::TT - 1) / F::TT;
  const long long DN = (long long)p.D * p.N, at = (long long)w.row * p.nchunks + w.piece;
  const auto tile_at = [&](int i) { return tbeg + (REV ? ntiles - 1 - i : i) * F::TT; };

  if (threadIdx.x < F::HALF) {
    const Lane<LN, NPT> q(p, w);
    const Both<NPT> A2 = load_decays(p, q);
    Both<NPT> h = load_both(p.A, q, p.N, false);
    for (int i = 0; i < ntiles; ++i) {
      tile_barrier();
      run_tile<LN, NPT, SEQ, true, REV>(p, w, q, s.tile[i & 1], A2, h, tile_at(i), tend, REV ? p.dfin : p.init);
    }
    store_both(p.cstate + at * DN, q, p.N, true, h);
    tile_barrier();
    return;
  }

  const Couple<LN, NPT> q(p, w);
  const int* seq = SEQ ? p.seq : nullptr;
  const float2 bias = params_of(p.bias, q.pd, q.on0, q.on1);
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + q.pd;
  // what drives the recurrence: u and B, or dout (gated) and C
  const T* v = REV ? static_cast<const T*>(p.dout) + (long long)w.row * p.L * p.D + q.pd
                   : static_cast<const T*>(p.u) + w.row * p.u_b + q.pd;
  const long long v_l = REV ? p.D : p.u_l;
  const T* z = static_cast<const T*>(p.z) + w.row * p.z_b + q.pd;
  const T* R = REV ? static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g
                   : static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const long long r_l = REV ? p.C_l : p.B_l;
  float2 sum = all2(0.f);
  Two<T> dd[F::TWOS], vv[F::TWOS], zz[F::TWOS];  // of the next tile, fetched an interval ahead
  Rows<T, F::NP, F::TT, F::HALF> rows;
  const auto fetch = [&](int i) {
    const int tn = tile_at(i);
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int tok = tn + q.tq + k * F::STEP;
      const bool in = tok < tend && in_sequence(seq, tok), on0 = in && q.on0, on1 = in && q.on1;
      dd[k] = load_two(delta + tok * p.delta_l, on0, on1, p.couples);
      vv[k] = load_two(v + tok * v_l, on0, on1, p.couples);
      if (REV) zz[k] = load_two(z + tok * p.z_l, on0 && p.z, on1 && p.z, p.couples);
    }
    rows.fetch(q.tid, R, r_l, tn, tend, seq, p.quads);
  };
  fetch(0);
  for (int i = 0; i < ntiles; ++i) {  // prepares tile i while tile i - 1 runs
    const int tn = tile_at(i);
    auto& tile = s.tile[i & 1];
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = q.tq + k * F::STEP, tok = tn + t;
      float2 dt = __fadd2_rn(two_f(dd[k]), bias), x = two_f(vv[k]);
      if (p.softplus) dt = softplus2(dt);
      if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
      if (REV && p.z) x = __fmul2_rn(x, silu2(two_f(zz[k])));
      if (!REV) x = __fmul2_rn(x, dt);
      sum = __fadd2_rn(sum, dt);
      *reinterpret_cast<float4*>(&tile.d[t * F::DT + q.pc]) = make_float4(dt.x, x.x, dt.y, x.y);
    }
    rows.put(q.tid, tile.B, R, r_l, tn, tend, p.N, seq, p.quads);
    if (i + 1 < ntiles) fetch(i + 1);
    tile_barrier();
  }
  // the couples' threads have the step sizes' sums, one token in STEP each
  float* part = s.tile[0].y;
  *reinterpret_cast<float2*>(&part[q.tq * F::DT + q.pc]) = sum;
  tile_barrier();
  if (q.tq == 0) {
#pragma unroll
    for (int j = 1; j < F::STEP; ++j) sum = __fadd2_rn(sum, *reinterpret_cast<const float2*>(&part[j * F::DT + q.pc]));
    if (q.on0) p.csum[at * p.D + q.pd] = sum.x;
    if (q.on1) p.csum[at * p.D + q.pd + 1] = sum.y;
  }
}

// Turns the pieces' end states into the states that enter them, in place. One thread per
// (row, channel, state).
template <bool REV>
__global__ void __launch_bounds__(256) scan_carry_kernel(const __grid_constant__ Params p) {
  const long long DN = (long long)p.D * p.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= DN * p.rows) return;
  const int row = i / DN;
  const long long i_dn = i - row * DN;
  const int d = i_dn / p.N;
  const float A2 = p.A[i_dn] * kLog2e;
  const float* edge = REV ? p.dfin : p.init;
  float h = edge && !p.seq ? edge[row * DN + i_dn] : 0.f;
  constexpr int AHEAD = 8;  // pieces read together: the chain through them is a few cycles each
  for (int k0 = 0; k0 < p.nchunks; k0 += AHEAD) {
    float own[AHEAD], sum[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      if (k0 + e >= p.nchunks) break;
      const long long at = (long long)row * p.nchunks + (REV ? p.nchunks - 1 - k0 - e : k0 + e);
      own[e] = p.cstate[at * DN + i_dn], sum[e] = p.csum[at * p.D + d];
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      if (k0 + e >= p.nchunks) break;
      const int c = REV ? p.nchunks - 1 - k0 - e : k0 + e;
      bool cut = false;
      if (p.seq) {  // a sequence that starts (ends) in the piece cuts what follows off from what came before
        const int t0 = c * p.chunk, t1 = min(p.L, t0 + p.chunk);
        cut = REV ? t1 >= p.L || p.seq[t1] != p.seq[t0] : t0 == 0 || p.seq[t0 - 1] != p.seq[t1 - 1];
      }
      p.cstate[((long long)row * p.nchunks + c) * DN + i_dn] = h;
      h = cut ? own[e] : fmaf(ex2(A2 * sum[e]), h, own[e]);
    }
  }
}

// ------------------------------------------------------------------------------ single token
struct StepParams {
  int rows, D, G, N, Dg, slots;
  const void *u, *delta, *B, *C, *z;
  long long u_b, delta_b, B_b, B_g, C_b, C_g, z_b, state_b;
  const float *A, *Dskip, *bias;
  int softplus;
  const int* index;  // each row's slot of the state, or NULL: row i has slot i
  float* state;      // [slots, D, N]
  void* out;         // [rows, D]
};

// A CTA has 128 / LN channels of ROWS rows, whose states are all on their way before the first is
// worked on: the state is read and written once, 8 N bytes a channel, and memory bounds it.
template <typename T, int LN, int NPT, int ROWS>
__global__ void __launch_bounds__(128) scan_step_kernel(const __grid_constant__ StepParams p) {
  constexpr int DT = 128 / LN;
  const int tid = threadIdx.x, nl = tid % LN, n0 = nl * NPT;
  const int tiles = (p.D + DT - 1) / DT;
  const int row0 = (int)(blockIdx.x / tiles) * ROWS, d = (int)(blockIdx.x % tiles) * DT + tid / LN;
  const bool on = d < p.D;
  int ok[ROWS];
  float h[ROWS][NPT], A2[NPT];
  float* state[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r;
    ok[r] = row < p.rows ? slot_state(p.index, row, p.slots) : 0;
    state[r] = p.state + (ok[r] > 0 ? (p.index ? p.index[row] : row) * p.state_b : 0);
    load_states<NPT>(state[r], d, n0, p.N, on && ok[r] > 0, h[r]);
  }
  load_states<NPT>(p.A, d, n0, p.N, on, A2);
  const float skip = on && p.Dskip ? p.Dskip[d] : 0.f, bias = on && p.bias ? p.bias[d] : 0.f;
  const int g = on ? d / p.Dg : 0;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r;
    if (row >= p.rows) break;
    T* out = static_cast<T*>(p.out) + (long long)row * p.D + d;
    if (ok[r] <= 0) {
      if (on && nl == 0) *out = from_f<T>(ok[r] < 0 ? __int_as_float(0x7fffffff) : 0.f);
      continue;
    }
    float y = 0.f, u = 0.f, z = 0.f;
    if (on) {
      u = to_f(static_cast<const T*>(p.u)[row * p.u_b + d]);
      if (p.z) z = to_f(static_cast<const T*>(p.z)[row * p.z_b + d]);
      float dt = to_f(static_cast<const T*>(p.delta)[row * p.delta_b + d]) + bias;
      if (p.softplus) dt = softplus(dt);
      const T* B = static_cast<const T*>(p.B) + row * p.B_b + g * p.B_g + n0;
      const T* C = static_cast<const T*>(p.C) + row * p.C_b + g * p.C_g + n0;
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        if (n0 + i < p.N) {
          h[r][i] = fmaf(ex2(fmaf(dt, A2[i] * kLog2e, kHalfStep)), h[r][i], dt * u * to_f(B[i]));
          y = fmaf(h[r][i], to_f(C[i]), y);
        }
      }
      store_states<NPT>(state[r], d, n0, p.N, true, h[r]);
    }
#pragma unroll
    for (int o = 1; o < LN; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (on && nl == 0) {
      y = fmaf(skip, u, y);
      if (p.z) y *= z * sigmoid(z);
      *out = from_f<T>(y);
    }
  }
}

// Sequence of each token from the sequences' ends: the last s with cu[s] <= t, if t < cu[s + 1].
__global__ void __launch_bounds__(256) sequence_index_kernel(int T, int S, const int* cu, int* seq) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  int lo = 0, hi = S;  // cu[lo] <= t < cu[hi], were cu[0] <= t < cu[S]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  seq[t] = cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

// ------------------------------------------------------------------------------ host
template <typename T>
static int launch_fwd(Params p, cudaStream_t st, const char* who) {
  return dispatch(p.N, [&](auto ln, auto npt) {
    using F = Fwd<decltype(ln)::value, decltype(npt)::value>;
    constexpr int LN = decltype(ln)::value, NPT = decltype(npt)::value;
    auto kernel = p.seq ? scan_fwd_kernel<T, LN, NPT, true> : scan_fwd_kernel<T, LN, NPT, false>;
    Params q = p;
    q.tiles = (p.Dg + F::DT - 1) / F::DT;
    const int rc = prepare_smem(kernel, sizeof(typename F::Smem), who);
    if (rc) return rc;
    const long long grid = (long long)q.tiles * q.G * q.nchunks * q.rows;
    TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
    kernel<<<(unsigned)grid, F::THREADS, sizeof(typename F::Smem), st>>>(q);
    return check_launch(who);
  });
}

template <typename T, bool REV>
static int launch_chunks(Params p, cudaStream_t st, const char* who) {
  return dispatch(p.N, [&](auto ln, auto npt) {
    using F = Fwd<decltype(ln)::value, decltype(npt)::value>;
    constexpr int LN = decltype(ln)::value, NPT = decltype(npt)::value;
    auto kernel = p.seq ? scan_chunk_kernel<T, LN, NPT, REV, true> : scan_chunk_kernel<T, LN, NPT, REV, false>;
    Params q = p;
    q.tiles = (p.Dg + F::DT - 1) / F::DT;
    int rc = prepare_smem(kernel, sizeof(typename F::Smem), who);
    if (rc) return rc;
    const long long grid = (long long)q.tiles * q.G * q.nchunks * q.rows;
    TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
    kernel<<<(unsigned)grid, F::THREADS, sizeof(typename F::Smem), st>>>(q);
    if ((rc = check_launch(who))) return rc;
    scan_carry_kernel<REV><<<(unsigned)(((long long)p.rows * p.D * p.N + 255) / 256), 256, 0, st>>>(q);
    return check_launch(who);
  });
}

int chunk_states(const Params& p, int dt, bool rev, cudaStream_t st, const char* who) {
  if (rev)
    return dt == DT_BF16  ? launch_chunks<__nv_bfloat16, true>(p, st, who)
           : dt == DT_F16 ? launch_chunks<__half, true>(p, st, who)
                          : launch_chunks<float, true>(p, st, who);
  return dt == DT_BF16  ? launch_chunks<__nv_bfloat16, false>(p, st, who)
         : dt == DT_F16 ? launch_chunks<__half, false>(p, st, who)
                        : launch_chunks<float, false>(p, st, who);
}

// Whether Rows::fetch may read B and C four states at a time.
bool quads(const Params& p, int dt) {
  const int elem = dt == DT_F32 ? 4 : 2;
  const Shape s = shape_of(p.N);
  if (p.N != s.LN * s.NPT) return false;
  for (const long long st : {p.B_b, p.B_l, p.B_g, p.C_b, p.C_l, p.C_g})
    if (st % 4) return false;
  return reinterpret_cast<uintptr_t>(p.B) % (4 * elem) == 0 && reinterpret_cast<uintptr_t>(p.C) % (4 * elem) == 0;
}

// Whether activations may be read and written two channels at a time.
bool couples(const Params& p, int dt) {
  const int two = dt == DT_F32 ? 8 : 4;
  if (p.Dg % 2) return false;
  for (const long long st : {p.u_b, p.u_l, p.delta_b, p.delta_l, p.z_b, p.z_l})
    if (st % 2) return false;
  for (const void* q : {p.u, p.delta, p.z, (const void*)p.out, p.dout, (const void*)p.du, (const void*)p.ddelta,
                        (const void*)p.dz})
    if (reinterpret_cast<uintptr_t>(q) % two) return false;
  return true;
}

// Tokens of a piece of the time axis, a multiple of 64 (tiles and kept states of every shape
// start on it), or L for one piece. Splitting costs a pass over the pieces first, `extra` of the
// main pass's time, about 128 tokens' worth of launches and 3 a piece; it pays where the `blocks` CTAs of
// whole rows leave SMs empty, or a last round of them nearly so. An SM runs `resident` CTAs at
// once; k of them take 0.4 + 0.6 k / resident of that time. Measured, 16 x 2048 x 1536 states
// of 16: backward 1.19 ms whole (384 CTAs on 296 places), 1.30 ms in 3 pieces, whose first pass
// alone takes 0.29 ms; 32 x 336 x 512 training 305 us in 3 or 4 pieces, 209 us whole; 1 x 8192 x 1024
// prompt 160 us in 128 pieces, 123 us in 26.
int piece_tokens(long long blocks, int L, int resident, float extra) {
  const long long sms = sm_count(), places = sms * resident;
  float best = 0.f;
  int tokens = L;
  const long long most = L / 64 < 1024 ? L / 64 : 1024;
  for (long long n = 1; n <= (most > 1 ? most : 1); ++n) {
    const int len = n == 1 ? L : (int)(((L + n - 1) / n + 63) / 64 * 64);
    const long long all = blocks * ((L + len - 1) / len), rest = all % places;
    float rounds = (float)(all / places);
    if (rest) rounds += 0.4f + 0.6f * (float)((rest + sms - 1) / sms) / resident;
    const float cost = n == 1 ? rounds * L : rounds * len * (1.f + extra) + 128.f + 3.f * n;
    if (n == 1 || cost < best) best = cost, tokens = len;
    if (all > 8 * places) break;
  }
  return tokens;
}

int check_sizes(const char* who, int rows, int L, int D, int G, int N, int dt) {
  TTT_REQUIRE(rows >= 1 && L >= 1 && D >= 1 && G >= 1 && N >= 1, TTT_ERR_SHAPE,
              "%s: sizes must be positive, got rows=%d L=%d D=%d G=%d N=%d", who, rows, L, D, G, N);
  TTT_REQUIRE(D % G == 0, TTT_ERR_SHAPE, "%s: %d channels do not divide into %d groups", who, D, G);
  TTT_REQUIRE(N <= kMaxStates, TTT_ERR_SHAPE, "%s: %d states per channel, at most %d", who, N, kMaxStates);
  TTT_REQUIRE((long long)rows * L < (1LL << 31) - 4096, TTT_ERR_SHAPE, "%s: %lld tokens are too many", who,
              (long long)rows * L);
  TTT_REQUIRE((long long)rows * D * N < (1LL << 38), TTT_ERR_SHAPE, "%s: too many states", who);
  TTT_REQUIRE(valid_dtype(dt), TTT_ERR_DTYPE, "%s: bad dtype code %d", who, dt);
  return TTT_OK;
}

// How the time axis is split, forwards or backwards: the CTAs have the same channels.
static int split(int rows, int L, int D, int G, int N, bool backward) {
  const int DT = 256 / shape_of(N).LN;
  const long long blocks = (long long)rows * G * ((D / G + DT - 1) / DT);
  const int NPT = shape_of(N).NPT;  // resident CTAs as the kernels' launch bounds have them
  return backward ? piece_tokens(blocks, L, NPT == 4 ? 2 : 1, 0.3f)
                  : piece_tokens(blocks, L, NPT == 4 ? 3 : NPT == 8 ? 2 : 1, 0.5f);
}
void plan_pieces(Params& p, bool backward) {
  p.chunk = split(p.rows, p.L, p.D, p.G, p.N, backward);
  p.nchunks = (p.L + p.chunk - 1) / p.chunk;
}
size_t piece_bytes(const Params& p) {
  return p.nchunks > 1 ? (size_t)p.rows * p.nchunks * p.D * (p.N + 1) * sizeof(float) : 0;
}
int plan_scratch(Params& p, void* scratch, size_t scratch_bytes, size_t extra, const char* who) {
  const size_t need = extra + piece_bytes(p);
  TTT_REQUIRE(!need || (scratch && scratch_bytes >= need), TTT_ERR_SCRATCH, "%s: scratch of %zu bytes needed, got %zu",
              who, need, scratch ? scratch_bytes : (size_t)0);
  if (p.nchunks > 1) {
    p.cstate = reinterpret_cast<float*>(static_cast<char*>(scratch) + extra);
    p.csum = p.cstate + (size_t)p.rows * p.nchunks * p.D * p.N;
  }
  return TTT_OK;
}

}  // namespace scan
}  // namespace ttt

using namespace ttt;

extern "C" size_t ttt_selective_scan_fwd_scratch_bytes(int rows, int L, int D, int G, int N) {
  if (rows < 1 || L < 1 || D < 1 || G < 1 || N < 1 || N > scan::kMaxStates || D % G) return 0;
  scan::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.G = G, p.N = N;
  scan::plan_pieces(p, false);
  return scan::piece_bytes(p);
}

extern "C" size_t ttt_selective_scan_saved_bytes(int rows, int L, int D, int N) {
  if (rows < 1 || L < 1 || D < 1 || N < 1 || N > scan::kMaxStates) return 0;
  const int every = scan::save_every(N);
  return (size_t)rows * ((L + every - 1) / every) * D * N * sizeof(float);
}

extern "C" int ttt_selective_scan_fwd(int rows, int L, int D, int G, int N, const void* u, const void* delta,
                                      const void* B, const void* C, const void* z, int dt, const long long* strides,
                                      const float* A, const float* Dskip, const float* delta_bias, int softplus,
                                      const int* seq, const float* init, float* fin, void* out, float* saved,
                                      void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "ttt_selective_scan_fwd";
  int rc = scan::check_sizes(who, rows, L, D, G, N, dt);
  if (rc) return rc;
  TTT_REQUIRE(u && delta && B && C && A && out && strides, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(!seq || rows == 1, TTT_ERR_SHAPE, "%s: packed sequences lie in one row, got %d", who, rows);
  scan::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.G = G, p.N = N, p.Dg = D / G;
  p.u = u, p.delta = delta, p.B = B, p.C = C, p.z = z;
  p.u_b = strides[0], p.u_l = strides[1], p.delta_b = strides[2], p.delta_l = strides[3];
  p.B_b = strides[4], p.B_l = strides[5], p.B_g = strides[6], p.C_b = strides[7], p.C_l = strides[8];
  p.C_g = strides[9], p.z_b = strides[10], p.z_l = strides[11];
  p.A = A, p.Dskip = Dskip, p.bias = delta_bias, p.softplus = softplus;
  p.seq = seq, p.init = init, p.fin = fin, p.out = out, p.hsave = saved;
  const int every = scan::save_every(N);
  p.nsave = (L + every - 1) / every;
  p.quads = scan::quads(p, dt), p.couples = scan::couples(p, dt);
  scan::plan_pieces(p, false);
  if ((rc = scan::plan_scratch(p, scratch, scratch_bytes, 0, who))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.nchunks > 1 && (rc = scan::chunk_states(p, dt, false, st, who))) return rc;
  return dt == DT_BF16  ? scan::launch_fwd<__nv_bfloat16>(p, st, who)
         : dt == DT_F16 ? scan::launch_fwd<__half>(p, st, who)
                        : scan::launch_fwd<float>(p, st, who);
}

extern "C" int ttt_selective_scan_step(int rows, int D, int G, int N, int slots, const void* u, const void* delta,
                                       const void* B, const void* C, const void* z, int dt, const long long* strides,
                                       const float* A, const float* Dskip, const float* delta_bias, int softplus,
                                       const int* index, float* state, void* out, void* stream) {
  const char* who = "ttt_selective_scan_step";
  int rc = scan::check_sizes(who, rows, 1, D, G, N, dt);
  if (rc) return rc;
  TTT_REQUIRE(u && delta && B && C && A && state && out && strides, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(slots >= 1 && (index || slots >= rows), TTT_ERR_SHAPE, "%s: %d states for %d rows", who, slots, rows);
  scan::StepParams p{};
  p.rows = rows, p.D = D, p.G = G, p.N = N, p.Dg = D / G, p.slots = slots;
  p.u = u, p.delta = delta, p.B = B, p.C = C, p.z = z;
  p.u_b = strides[0], p.delta_b = strides[1], p.B_b = strides[2], p.B_g = strides[3], p.C_b = strides[4];
  p.C_g = strides[5], p.z_b = strides[6], p.state_b = strides[7];
  p.A = A, p.Dskip = Dskip, p.bias = delta_bias, p.softplus = softplus, p.index = index, p.state = state, p.out = out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return scan::dispatch(N, [&](auto ln, auto npt) {
    constexpr int LN = decltype(ln)::value, NPT = decltype(npt)::value, DT = 128 / LN;
    // four rows a CTA once one row each would be over 16 CTAs an SM: fewer, with more loads in flight
    const long long tiles = (D + DT - 1) / DT;
    const int each = tiles * rows > 16LL * scan::sm_count() ? 4 : 1;
    const long long grid = tiles * ((rows + each - 1) / each);
    TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
    const auto go = [&](auto zero) {
      using T = decltype(zero);
      auto kernel = each == 4 ? scan::scan_step_kernel<T, LN, NPT, 4> : scan::scan_step_kernel<T, LN, NPT, 1>;
      kernel<<<(unsigned)grid, 128, 0, st>>>(p);
    };
    if (dt == DT_BF16) go(__nv_bfloat16{});
    else if (dt == DT_F16) go(__half{});
    else go(float{});
    return check_launch(who);
  });
}

extern "C" int ttt_sequence_index(int T, int S, const int* cu_seqlens, int* seq, void* stream) {
  const char* who = "ttt_sequence_index";
  TTT_REQUIRE(cu_seqlens && seq, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(T >= 1 && S >= 1 && T < (1 << 30), TTT_ERR_SHAPE, "%s: bad sizes T=%d S=%d", who, T, S);
  scan::sequence_index_kernel<<<(T + 255) / 256, 256, 0, static_cast<cudaStream_t>(stream)>>>(T, S, cu_seqlens, seq);
  return check_launch(who);
}
