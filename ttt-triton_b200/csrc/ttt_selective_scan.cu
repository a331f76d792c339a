// Selective state space scan, forward: prompts, packed prompts and the training forward, and
// the single-token step. The recurrence is in selective_scan.cuh.
//
// A channel's N states are split over LN threads, NPT in each, and stay in registers while the
// CTA walks the time axis tile by tile: a tile's step sizes and inputs are worked out once per
// (token, channel) into shared memory, then every thread runs its states through the tile's
// tokens, then the threads add the partial outputs of their channel, apply the skip and the
// gate and write. One exponential per (token, channel, state) is what bounds it.
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
  static constexpr int THREADS = 128, WARPS = THREADS / 32;
  static constexpr int DT = THREADS / LN;            // channels of a CTA
  static constexpr int NP = LN * NPT;                // states, padded
  static constexpr int TT = LN >= 4 ? 32 : 8 * LN;   // tokens of a tile
  static constexpr int RUN = 8;                      // tokens unrolled
  static constexpr int TWOS = TT * DT / 2 / THREADS; // couples of channels of a thread, one token each
  static constexpr int STEP = 2 * LN;                // tokens between them
  struct Smem {
    float B[TT * NP], C[TT * NP];
    float4 d[TT * DT];      // step size twice, step size * input twice: operands of paired arithmetic
    float y[TT * THREADS];  // partial outputs
    unsigned dt_max[WARPS], A_max[WARPS];
    SeqMask m;
  };
};

// What a thread holds: channel d and states n0 .. in the recurrence; channels pd, pd + 1, and
// tokens tq, tq + STEP, .. of a tile, in the element-wise passes.
template <int LN, int NPT>
struct Lane {
  int n0, cl, d, tq, pc, pd;
  bool on, on0, on1;
  __device__ __forceinline__ Lane(const Params& p, const Where& w) {
    using F = Fwd<LN, NPT>;
    const int tid = threadIdx.x;
    n0 = tid % LN * NPT, cl = tid / LN;
    pc = tid % (F::DT / 2) * 2, tq = tid / (F::DT / 2);
    d = w.g * p.Dg + w.d0 + cl, pd = w.g * p.Dg + w.d0 + pc;
    on = w.d0 + cl < p.Dg, on0 = w.d0 + pc < p.Dg, on1 = w.d0 + pc + 1 < p.Dg;
  }
};
// One token of the recurrence for NPT states; POLY: this token's share of the decays goes to
// the multiply-add pipes (3 pairs in 8, see pow2_poly).
template <int NPT, bool POLY>
__device__ __forceinline__ void advance(Pairs<NPT>& h, const Pairs<NPT>& A2, const float4 dd, const float* Brow,
                                        int t) {
  const float2 dt = make_float2(dd.x, dd.y), dtu = make_float2(dd.z, dd.w);
  const Pairs<NPT> B = row_pairs<NPT>(Brow);
#pragma unroll
  for (int j = 0; j < NPT / 2; ++j) {
    const int k = (t * (NPT / 2) + j) % 8;
    const float2 a = POLY && (k == 1 || k == 4 || k == 6) ? pow2_poly(dt, A2.v[j]) : pow2_unit(dt, A2.v[j]);
    h.v[j] = __ffma2_rn(a, h.v[j], __fmul2_rn(dtu, B.v[j]));
  }
}

template <typename T, int LN, int NPT, bool SEQ>
__global__ void __launch_bounds__(128) scan_fwd_kernel(const __grid_constant__ Params p) {
  using F = Fwd<LN, NPT>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const Lane<LN, NPT> q(p, w);
  const int tid = threadIdx.x;
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const long long DN = (long long)p.D * p.N;
  const int* seq = SEQ ? p.seq : nullptr;

  float hs[NPT];
  load_states<NPT>(p.A, q.d, q.n0, p.N, q.on, hs);
  unsigned am = 0;
#pragma unroll
  for (int i = 0; i < NPT; i += 2) {
    hs[i] *= kLog2e, hs[i + 1] *= kLog2e;
    am = max_bits(am, make_float2(hs[i], hs[i + 1]));
  }
  am = __reduce_max_sync(0xffffffffu, am);
  if (tid % 32 == 0) s.A_max[tid / 32] = am;
  const Pairs<NPT> A2 = pairs_of<NPT>(hs);
  if (p.nchunks > 1)
    load_states<NPT>(p.cstate + ((long long)w.row * p.nchunks + w.piece) * DN, q.d, q.n0, p.N, q.on, hs);
  else
    load_states<NPT>(p.init + w.row * DN, q.d, q.n0, p.N, q.on && p.init && !SEQ, hs);
  Pairs<NPT> h = pairs_of<NPT>(hs);
  const float2 skip = params_of(p.Dskip, q.pd, q.on0, q.on1), bias = params_of(p.bias, q.pd, q.on0, q.on1);
  const long long first = tbeg + q.tq;
  const T* u = static_cast<const T*>(p.u) + w.row * p.u_b + first * p.u_l + q.pd;
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + first * p.delta_l + q.pd;
  const T* z = static_cast<const T*>(p.z) + w.row * p.z_b + first * p.z_l + q.pd;
  const T* B = static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const T* C = static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g;
  T* out = static_cast<T*>(p.out) + ((long long)w.row * p.L + first) * p.D + q.pd;
  const long long u_step = F::STEP * p.u_l, delta_step = F::STEP * p.delta_l, z_step = F::STEP * p.z_l;
  const long long out_step = (long long)F::STEP * p.D;
  const int every = 32 / NPT;

  for (int t0 = tbeg; t0 < tend; t0 += F::TT) {
    Two<T> uu[F::TWOS], zz[F::TWOS], dd[F::TWOS];
    if (SEQ) stage_masks<F::TT>(&s.m, p.seq, t0, tend, p.L);
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int tok = t0 + q.tq + k * F::STEP;
      const bool in = tok < tend && in_sequence(seq, tok), on0 = in && q.on0, on1 = in && q.on1;
      dd[k] = load_two(delta, on0, on1, p.couples), uu[k] = load_two(u, on0, on1, p.couples);
      zz[k] = load_two(z, on0 && p.z, on1 && p.z, p.couples);
      delta += delta_step, u += u_step, z += z_step;
    }
    stage_rows<T, F::NP, F::TT, F::THREADS>(s.B, B, p.B_l, t0, tend, p.N, seq, p.quads);
    stage_rows<T, F::NP, F::TT, F::THREADS>(s.C, C, p.C_l, t0, tend, p.N, seq, p.quads);
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = q.tq + k * F::STEP, tok = t0 + t;
      float2 dt = __fadd2_rn(two_f(dd[k]), bias);
      if (p.softplus) dt = softplus2(dt);
      if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
      const float2 x = __fmul2_rn(dt, two_f(uu[k]));
      m = max_bits(m, dt);
      s.d[t * F::DT + q.pc] = make_float4(dt.x, dt.x, x.x, x.x);
      s.d[t * F::DT + q.pc + 1] = make_float4(dt.y, dt.y, x.y, x.y);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (tid % 32 == 0) s.dt_max[tid / 32] = m;
    __syncthreads();
    const bool poly = max_of(s.dt_max) * max_of(s.A_max) < kPolyRange;

#pragma unroll 1
    for (int r = 0; r < F::TT && t0 + r < tend; r += F::RUN) {
      if (p.hsave && (t0 + r) % every == 0) {
        unpair(h, hs);
        store_states<NPT>(p.hsave + ((long long)w.row * p.nsave + (t0 + r) / every) * DN, q.d, q.n0, p.N, q.on, hs);
      }
      const bool slow =
          t0 + r + F::RUN > tend || (SEQ && ((s.m.start | s.m.end) >> r & 0xff)) || (p.hsave && every < F::RUN);
      const auto tokens = [&](auto use_poly, auto checks) {
#pragma unroll
        for (int k = 0; k < F::RUN; ++k) {
          const int t = r + k;
          if constexpr (decltype(checks)::value) {
            if (t0 + t >= tend) break;
            if (p.hsave && k && (t0 + t) % every == 0) {
              unpair(h, hs);
              store_states<NPT>(p.hsave + ((long long)w.row * p.nsave + (t0 + t) / every) * DN, q.d, q.n0, p.N, q.on,
                                hs);
            }
            if (SEQ && (s.m.start >> t & 1)) {
              const int sq = p.seq[t0 + t];
              load_states<NPT>(p.init + sq * DN, q.d, q.n0, p.N, q.on && sq >= 0 && p.init, hs);
              h = pairs_of<NPT>(hs);
            }
          }
          advance<NPT, decltype(use_poly)::value>(h, A2, s.d[t * F::DT + q.cl], s.B + t * F::NP + q.n0, k);
          const Pairs<NPT> C2 = row_pairs<NPT>(s.C + t * F::NP + q.n0);
          float2 y = __fmul2_rn(h.v[0], C2.v[0]);
#pragma unroll
          for (int j = 1; j < NPT / 2; ++j) y = __ffma2_rn(h.v[j], C2.v[j], y);
          s.y[t * F::THREADS + tid] = y.x + y.y;
          if constexpr (decltype(checks)::value) {
            if (SEQ && p.fin && (s.m.end >> t & 1)) {
              const int sq = p.seq[t0 + t];
              unpair(h, hs);
              store_states<NPT>(p.fin + sq * DN, q.d, q.n0, p.N, q.on && sq >= 0, hs);
            }
          }
        }
      };
      if (slow) tokens(std::false_type{}, std::true_type{});
      else if (poly) tokens(std::true_type{}, std::false_type{});
      else tokens(std::false_type{}, std::false_type{});
    }
    __syncthreads();

#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = q.tq + k * F::STEP, tok = t0 + t;
      float2 y = __ffma2_rn(skip, two_f(uu[k]), state_sums<LN>(s.y + t * F::THREADS + q.pc * LN));
      if (p.z) y = __fmul2_rn(y, silu2(two_f(zz[k])));
      if (SEQ && !(s.m.in >> t & 1)) y = all2(0.f);  // a token of no sequence
      store_two(out, y, q.on0 && tok < tend, q.on1 && tok < tend, p.couples);
      out += out_step;
    }
    if (SEQ) __syncthreads();  // the masks are written again
  }
  if (!SEQ && p.fin && tend == p.L) {
    unpair(h, hs);
    store_states<NPT>(p.fin + w.row * DN, q.d, q.n0, p.N, q.on, hs);
  }
}

// A piece's end state from zero (REV: the carry that leaves its first token from zero at its
// last), and the sum of its step sizes.
template <typename T, int LN, int NPT, bool REV, bool SEQ>
__global__ void __launch_bounds__(128) scan_chunk_kernel(const __grid_constant__ Params p) {
  using F = Fwd<LN, NPT>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const Lane<LN, NPT> q(p, w);
  const int tid = threadIdx.x;
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const long long DN = (long long)p.D * p.N;
  const int* seq = SEQ ? p.seq : nullptr;

  float hs[NPT], sum = 0.f;
  load_states<NPT>(p.A, q.d, q.n0, p.N, q.on, hs);
  unsigned am = 0;
#pragma unroll
  for (int i = 0; i < NPT; i += 2) {
    hs[i] *= kLog2e, hs[i + 1] *= kLog2e;
    am = max_bits(am, make_float2(hs[i], hs[i + 1]));
  }
  am = __reduce_max_sync(0xffffffffu, am);
  if (tid % 32 == 0) s.A_max[tid / 32] = am;
  const Pairs<NPT> A2 = pairs_of<NPT>(hs);
  Pairs<NPT> h;
#pragma unroll
  for (int j = 0; j < NPT / 2; ++j) h.v[j] = make_float2(0.f, 0.f);
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
  const float* edge = REV ? p.dfin : p.init;

  const int ntiles = (tend - tbeg + F::TT - 1) / F::TT;
  for (int k0 = 0; k0 < ntiles; ++k0) {
    const int t0 = tbeg + (REV ? ntiles - 1 - k0 : k0) * F::TT;
    if (SEQ) stage_masks<F::TT>(&s.m, p.seq, t0, tend, p.L);
    Two<T> dd[F::TWOS], vv[F::TWOS], zz[F::TWOS];
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int tok = t0 + q.tq + k * F::STEP;
      const bool in = tok < tend && in_sequence(seq, tok), on0 = in && q.on0, on1 = in && q.on1;
      dd[k] = load_two(delta + tok * p.delta_l, on0, on1, p.couples);
      vv[k] = load_two(v + tok * v_l, on0, on1, p.couples);
      if (REV) zz[k] = load_two(z + tok * p.z_l, on0 && p.z, on1 && p.z, p.couples);
    }
    stage_rows<T, F::NP, F::TT, F::THREADS>(s.B, R, r_l, t0, tend, p.N, seq, p.quads);
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = q.tq + k * F::STEP, tok = t0 + t;
      float2 dt = __fadd2_rn(two_f(dd[k]), bias), x = two_f(vv[k]);
      if (p.softplus) dt = softplus2(dt);
      if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
      if (REV && p.z) x = __fmul2_rn(x, silu2(two_f(zz[k])));
      if (!REV) x = __fmul2_rn(x, dt);
      m = max_bits(m, dt);
      s.d[t * F::DT + q.pc] = make_float4(dt.x, dt.x, x.x, x.x);
      s.d[t * F::DT + q.pc + 1] = make_float4(dt.y, dt.y, x.y, x.y);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (tid % 32 == 0) s.dt_max[tid / 32] = m;
    __syncthreads();
    const bool poly = max_of(s.dt_max) * max_of(s.A_max) < kPolyRange;

#pragma unroll 1
    for (int r0 = 0; r0 < F::TT; r0 += F::RUN) {
      const int r = REV ? F::TT - F::RUN - r0 : r0;
      if (t0 + r >= tend) continue;
      const auto tokens = [&](auto use_poly, auto checks) {
#pragma unroll
        for (int k = 0; k < F::RUN; ++k) {
          const int t = r + (REV ? F::RUN - 1 - k : k);
          if constexpr (decltype(checks)::value) {
            if (t0 + t >= tend) continue;
            if (SEQ && ((REV ? s.m.end : s.m.start) >> t & 1)) {
              const int sq = p.seq[t0 + t];
              load_states<NPT>(edge + sq * DN, q.d, q.n0, p.N, q.on && sq >= 0 && edge, hs);
              h = pairs_of<NPT>(hs);
            }
          }
          const float4 dd4 = s.d[t * F::DT + q.cl];
          const float* row = s.B + t * F::NP + q.n0;
          sum += dd4.x;
          if constexpr (REV) {
            const Pairs<NPT> R2 = row_pairs<NPT>(row);
            const float2 dt = make_float2(dd4.x, dd4.y), x = make_float2(dd4.z, dd4.w);
#pragma unroll
            for (int j = 0; j < NPT / 2; ++j) {
              const int i = (k * (NPT / 2) + j) % 8;
              const float2 a = decltype(use_poly)::value && (i == 1 || i == 4 || i == 6) ? pow2_poly(dt, A2.v[j])
                                                                                         : pow2_unit(dt, A2.v[j]);
              h.v[j] = __fmul2_rn(a, __ffma2_rn(x, R2.v[j], h.v[j]));
            }
          } else {
            advance<NPT, decltype(use_poly)::value>(h, A2, dd4, row, k);
          }
        }
      };
      if (t0 + r + F::RUN > tend || (SEQ && ((REV ? s.m.end : s.m.start) >> r & 0xff))) tokens(std::false_type{}, std::true_type{});
      else if (poly) tokens(std::true_type{}, std::false_type{});
      else tokens(std::false_type{}, std::false_type{});
    }
    __syncthreads();
  }
  const long long at = (long long)w.row * p.nchunks + w.piece;
  unpair(h, hs);
  store_states<NPT>(p.cstate + at * DN, q.d, q.n0, p.N, q.on, hs);
  if (q.on && tid % LN == 0) p.csum[at * p.D + q.d] = sum;
}

// Turns the pieces' end states into the states that enter them, in place. One thread per
// (row, channel, state).
template <bool REV>
__global__ void __launch_bounds__(256) scan_carry_kernel(const __grid_constant__ Params p) {
  const long long DN = (long long)p.D * p.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= DN * p.rows) return;
  const int row = i / DN;
  const long long e = i - row * DN;
  const int d = e / p.N;
  const float A2 = p.A[e] * kLog2e;
  const float* edge = REV ? p.dfin : p.init;
  float h = edge && !p.seq ? edge[row * DN + e] : 0.f;
  for (int k = 0; k < p.nchunks; ++k) {
    const int c = REV ? p.nchunks - 1 - k : k;
    const long long at = (long long)row * p.nchunks + c;
    bool cut = false;
    if (p.seq) {  // a sequence that starts (ends) in the piece cuts what follows off from what came before
      const int t0 = c * p.chunk, t1 = min(p.L, t0 + p.chunk);
      cut = REV ? t1 >= p.L || p.seq[t1] != p.seq[t0] : t0 == 0 || p.seq[t0 - 1] != p.seq[t1 - 1];
    }
    float* q = p.cstate + at * DN + e;
    const float own = *q;
    *q = h;
    h = cut ? own : fmaf(ex2(A2 * p.csum[at * p.D + d]), h, own);
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

template <typename T, int LN, int NPT>
__global__ void __launch_bounds__(128) scan_step_kernel(const __grid_constant__ StepParams p) {
  constexpr int DT = 128 / LN;
  const int tid = threadIdx.x, nl = tid % LN, n0 = nl * NPT;
  const int tiles = (p.D + DT - 1) / DT;
  const int row = blockIdx.x / tiles, d = (blockIdx.x - row * tiles) * DT + tid / LN;
  const bool on = d < p.D;
  const int ok = slot_state(p.index, row, p.slots);
  if (ok <= 0) {
    if (on && nl == 0)
      static_cast<T*>(p.out)[(long long)row * p.D + d] = from_f<T>(ok < 0 ? __int_as_float(0x7fffffff) : 0.f);
    return;
  }
  float y = 0.f, u = 0.f, z = 0.f;
  if (on) {
    float* state = p.state + (long long)(p.index ? p.index[row] : row) * p.state_b;
    const int g = d / p.Dg;
    u = to_f(static_cast<const T*>(p.u)[row * p.u_b + d]);
    if (p.z) z = to_f(static_cast<const T*>(p.z)[row * p.z_b + d]);
    const float dt = p.softplus
                         ? softplus(to_f(static_cast<const T*>(p.delta)[row * p.delta_b + d]) + (p.bias ? p.bias[d] : 0.f))
                         : to_f(static_cast<const T*>(p.delta)[row * p.delta_b + d]) + (p.bias ? p.bias[d] : 0.f);
    const T* B = static_cast<const T*>(p.B) + row * p.B_b + g * p.B_g;
    const T* C = static_cast<const T*>(p.C) + row * p.C_b + g * p.C_g;
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      const int n = n0 + i;
      if (n < p.N) {
        const long long e = (long long)d * p.N + n;
        const float h = fmaf(ex2(dt * (p.A[e] * kLog2e)), state[e], dt * u * to_f(B[n]));
        state[e] = h;
        y = fmaf(h, to_f(C[n]), y);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < LN; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (on && nl == 0) {
    if (p.Dskip) y = fmaf(p.Dskip[d], u, y);
    if (p.z) y *= z * sigmoid(z);
    static_cast<T*>(p.out)[(long long)row * p.D + d] = from_f<T>(y);
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

// Whether stage_rows may read B and C four states at a time.
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

// Pieces of the time axis: as many as bring the device about two full waves of warps, no
// piece under 64 tokens.
int pieces(int rows, int L, int D, int N) {
  const Shape s = shape_of(N);
  const long long warps = ((long long)rows * D * s.LN + 31) / 32, want = (long long)sm_count() * 32;
  if (warps >= want / 2 || L < 256) return 1;
  long long n = (want + warps - 1) / warps;
  if (n > L / 64) n = L / 64;
  return n < 1 ? 1 : (int)n;
}
// Tokens of a piece: a multiple of 64, so that tiles and saved states of every shape start on it.
int piece_tokens(int L, int n) { return ((L + n - 1) / n + 63) / 64 * 64; }

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

// Splits the time axis and lays the scratch out; `extra` bytes of the caller come first.
int plan(Params& p, void* scratch, size_t scratch_bytes, size_t extra, const char* who) {
  const int n = pieces(p.rows, p.L, p.D, p.N);
  p.chunk = n > 1 ? piece_tokens(p.L, n) : p.L;
  p.nchunks = (p.L + p.chunk - 1) / p.chunk;
  const size_t states = (size_t)p.rows * p.nchunks * p.D;
  const size_t need = extra + (p.nchunks > 1 ? states * (p.N + 1) * sizeof(float) : 0);
  TTT_REQUIRE(!need || (scratch && scratch_bytes >= need), TTT_ERR_SCRATCH, "%s: scratch of %zu bytes needed, got %zu",
              who, need, scratch ? scratch_bytes : (size_t)0);
  if (p.nchunks > 1) {
    p.cstate = reinterpret_cast<float*>(static_cast<char*>(scratch) + extra);
    p.csum = p.cstate + states * p.N;
  }
  return TTT_OK;
}
size_t plan_bytes(int rows, int L, int D, int N) {
  const int n = pieces(rows, L, D, N);
  if (n <= 1) return 0;
  const int chunk = piece_tokens(L, n), nchunks = (L + chunk - 1) / chunk;
  return nchunks > 1 ? (size_t)rows * nchunks * D * (N + 1) * sizeof(float) : 0;
}

}  // namespace scan
}  // namespace ttt

using namespace ttt;

extern "C" size_t ttt_selective_scan_fwd_scratch_bytes(int rows, int L, int D, int G, int N) {
  if (rows < 1 || L < 1 || D < 1 || G < 1 || N < 1 || N > scan::kMaxStates) return 0;
  return scan::plan_bytes(rows, L, D, N);
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
  if ((rc = scan::plan(p, scratch, scratch_bytes, 0, who))) return rc;
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
    const long long grid = (long long)((D + DT - 1) / DT) * rows;
    TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
    if (dt == DT_BF16) scan::scan_step_kernel<__nv_bfloat16, LN, NPT><<<(unsigned)grid, 128, 0, st>>>(p);
    else if (dt == DT_F16) scan::scan_step_kernel<__half, LN, NPT><<<(unsigned)grid, 128, 0, st>>>(p);
    else scan::scan_step_kernel<float, LN, NPT><<<(unsigned)grid, 128, 0, st>>>(p);
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
