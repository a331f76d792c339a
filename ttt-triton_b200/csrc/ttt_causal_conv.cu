// Short causal convolution along the sequence, per channel, with K = 2 .. 4 taps:
//
//   p[t] = bias + sum_k w[k] x[t - K + 1 + k],  y = p or p sigmoid(p)
//
// Rows before a sequence's first token are its initial state's K - 1 rows, or zero; the final
// state is its last K - 1 rows. It moves every value once in and once out with a handful of
// operations each, so memory is its floor: a thread holds VEC adjacent channels (a vector load
// per token), walks a run of tokens with the last K - 1 rows in registers, and loads several
// tokens together; a warp covers 32 adjacent vectors of one run, a block 8 runs. Measured, 32 x
// 4096 x 1024 bf16, K = 4, silu: 150 us forward (3.6 TB/s), 240 us backward (3.4 TB/s). The latency of
// those loads bounds it: 14 warps an SM issue 1.1 to 1.3 instructions a clock and wait for global
// memory most of the rest, as nothing is on its way while a block of tokens is worked on.
//
// Backward, dp = dy act'(p): dx[t] = sum_k w[k] dp[t + K - 1 - k], dw[k] = sum dp x, db = sum
// dp. One walk forward in time: each dp is added to the gradients of the K rows that it
// reaches, which are in registers, and the oldest is then complete. Blocks write partial dw
// and db, which are added in a fixed order.
#include "scan_common.cuh"

namespace ttt {
namespace conv {

using scan::from_f;
using scan::to_f;

constexpr int kWarps = 8;

struct Params {
  int rows, L, D, act;
  int run, runs;           // tokens of a run, runs of a row
  long long x_b, x_l;      // element strides of x
  const void* x;
  const float *w, *b;      // [D, K], [D] or NULL
  const int* seq;          // packed rows: each token's sequence, else NULL
  const void* init;        // [sequences, K - 1, D] or NULL
  void* fin;
  void* y;                 // [rows, L, D]
  const void *dy, *dfin;   // [rows, L, D], [sequences, K - 1, D] or NULL
  void *dx, *dinit;
  float* part;             // [blocks of runs, D * (K + 1)]: dw | db
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
// VEC channels' values as pairs (the last one's second is unused where VEC is 1).
template <int VEC>
struct Vals {
  static constexpr int H = (VEC + 1) / 2;
  float2 v[H];
};
template <typename T, int VEC>
__device__ __forceinline__ Vals<VEC> unpack(const Pack<T, VEC>& r) {
  Vals<VEC> x;
#pragma unroll
  for (int j = 0; j < Vals<VEC>::H; ++j)
    x.v[j] = make_float2(to_f(r.v[2 * j]), 2 * j + 1 < VEC ? to_f(r.v[(2 * j + 1) % VEC]) : 0.f);
  return x;
}
template <int VEC>
__device__ __forceinline__ Vals<VEC> zeros() {
  Vals<VEC> x;
#pragma unroll
  for (int j = 0; j < Vals<VEC>::H; ++j) x.v[j] = make_float2(0.f, 0.f);
  return x;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load(const void* base, long long at) {
  return *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(base) + at);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(void* base, long long at, const Vals<VEC>& x) {
  Pack<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = from_f<T>(e % 2 ? x.v[e / 2].y : x.v[e / 2].x);
  *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(base) + at) = r;
}
template <int VEC>
__device__ __forceinline__ Vals<VEC> fma_of(const Vals<VEC>& a, const Vals<VEC>& b, const Vals<VEC>& c) {
  Vals<VEC> r;
#pragma unroll
  for (int j = 0; j < Vals<VEC>::H; ++j) r.v[j] = __ffma2_rn(a.v[j], b.v[j], c.v[j]);
  return r;
}
__device__ __forceinline__ float2 sigmoid2(float2 x) {
  const float2 m = __fmul2_rn(x, make_float2(-scan::kLog2e, -scan::kLog2e));
  const float2 e = __fadd2_rn(make_float2(scan::ex2(m.x), scan::ex2(m.y)), make_float2(1.f, 1.f));
  return make_float2(scan::rcp(e.x), scan::rcp(e.y));
}

// The channels' weights, tap 0 on the oldest row, and bias.
template <int K, int VEC>
struct Taps {
  Vals<VEC> w[K], b;
  __device__ __forceinline__ Taps(const Params& p, int d) {
#pragma unroll
    for (int j = 0; j < Vals<VEC>::H; ++j) {
      const int d0 = d + 2 * j, d1 = d + (2 * j + 1 < VEC ? 2 * j + 1 : 2 * j);
#pragma unroll
      for (int k = 0; k < K; ++k) w[k].v[j] = make_float2(p.w[(long long)d0 * K + k], p.w[(long long)d1 * K + k]);
      b.v[j] = make_float2(p.b ? p.b[d0] : 0.f, p.b ? p.b[d1] : 0.f);
    }
  }
  // bias + sum of taps over x and the K - 1 rows before it, hist[0] the nearest
  __device__ __forceinline__ Vals<VEC> at(const Vals<VEC>& x, const Vals<VEC> (&hist)[K - 1]) const {
    Vals<VEC> q = fma_of(w[K - 1], x, b);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) q = fma_of(w[K - 2 - j], hist[j], q);
    return q;
  }
};
template <int K, int VEC>
__device__ __forceinline__ void push(Vals<VEC> (&hist)[K - 1], const Vals<VEC>& x) {
#pragma unroll
  for (int j = K - 2; j > 0; --j) hist[j] = hist[j - 1];
  hist[0] = x;
}

struct At {
  int row, t0, t1;
  bool on;
};
__device__ __forceinline__ At run_of(const Params& p, long long id) {
  At a;
  a.on = id < (long long)p.rows * p.runs;
  a.row = a.on ? (int)(id / p.runs) : 0;
  a.t0 = a.on ? (int)(id - (long long)a.row * p.runs) * p.run : 0;
  a.t1 = a.on ? min(p.L, a.t0 + p.run) : 0;
  return a;
}
template <bool SEQ>
__device__ __forceinline__ bool starts(const Params& p, int t) {
  return SEQ ? scan::seq_starts(p.seq, t) : t == 0;
}
template <bool SEQ>
__device__ __forceinline__ bool ends(const Params& p, int t) {
  return SEQ ? scan::seq_ends(p.seq, t, p.L) : t == p.L - 1;
}
// Whether none of the tokens t .. t + U - 1 starts or ends a sequence or belongs to none.
template <int U, bool SEQ>
__device__ __forceinline__ bool plain(const Params& p, int t) {
  if (!SEQ) return t > 0 && t + U < p.L;
  const int i = t + (threadIdx.x & 31);
  const bool bad = (threadIdx.x & 31) < U && (i >= p.L || p.seq[i] < 0 || scan::seq_starts(p.seq, i) || scan::seq_ends(p.seq, i, p.L));
  return !__any_sync(0xffffffffu, bad);
}

// The K - 1 rows before a sequence's first token.
template <typename T, int K, int VEC>
__device__ __forceinline__ void initial_rows(const Params& p, int s, int d, Vals<VEC> (&hist)[K - 1]) {
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    hist[j] = p.init && s >= 0 ? unpack<T, VEC>(load<T, VEC>(p.init, ((long long)s * (K - 1) + K - 2 - j) * p.D + d))
                               : zeros<VEC>();
}
// The rows before token t0 > 0 of a run, of its sequence. Returns the sequence's first token if that
// is among them, else -K.
template <typename T, int K, int VEC, bool SEQ>
__device__ __forceinline__ int rows_before(const Params& p, const T* x, int t0, int d, Vals<VEC> (&hist)[K - 1]) {
  int first = -K;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) hist[j] = zeros<VEC>();
  for (int t = max(0, t0 - (K - 1)); t < t0; ++t) {
    if (SEQ && starts<SEQ>(p, t)) initial_rows<T, K, VEC>(p, p.seq[t], d, hist), first = t;
    push<K, VEC>(hist, unpack<T, VEC>(load<T, VEC>(x, t * p.x_l)));
  }
  return first;
}

template <typename T, int K, int VEC, bool SEQ>
__global__ void __launch_bounds__(kWarps * 32) conv_fwd_kernel(const __grid_constant__ Params p) {
  constexpr int U = 8;  // tokens loaded together
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = (p.D / VEC + 31) / 32;
  const long long blk = blockIdx.x / groups;
  int d = ((int)(blockIdx.x - blk * groups) * 32 + lane) * VEC;
  const At a = run_of(p, blk * kWarps + warp);
  if (!a.on) return;
  const bool on = d < p.D;
  if (!on) d = 0;  // the lanes past the row stay for the warp's votes and write nothing
  const Taps<K, VEC> taps(p, d);
  const T* x = static_cast<const T*>(p.x) + a.row * p.x_b + d;
  T* y = static_cast<T*>(p.y) + (long long)a.row * p.L * p.D + d;
  Vals<VEC> hist[K - 1];
  rows_before<T, K, VEC, SEQ>(p, x, a.t0, d, hist);
  const auto output = [&](const Vals<VEC>& v) {
    Vals<VEC> q = taps.at(v, hist);
    if (p.act)
#pragma unroll
      for (int j = 0; j < Vals<VEC>::H; ++j) q.v[j] = __fmul2_rn(q.v[j], sigmoid2(q.v[j]));
    push<K, VEC>(hist, v);
    return q;
  };
  for (int t = a.t0; t < a.t1;) {
    if (t + U <= a.t1 && plain<U, SEQ>(p, t)) {
      Pack<T, VEC> in[U];
#pragma unroll
      for (int i = 0; i < U; ++i) in[i] = load<T, VEC>(x, (t + i) * p.x_l);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const Vals<VEC> q = output(unpack<T, VEC>(in[i]));
        if (on) store<T, VEC>(y, (long long)(t + i) * p.D, q);
      }
      t += U;
      continue;
    }
    for (const int stop = min(t + U, a.t1); t < stop; ++t) {
      const int s = SEQ ? p.seq[t] : a.row;
      if (starts<SEQ>(p, t)) initial_rows<T, K, VEC>(p, s, d, hist);
      Vals<VEC> q = output(unpack<T, VEC>(load<T, VEC>(x, t * p.x_l)));
      if (s < 0) q = zeros<VEC>();
      if (on) store<T, VEC>(y, (long long)t * p.D, q);
      if (on && p.fin && s >= 0 && ends<SEQ>(p, t))
#pragma unroll
        for (int j = 0; j < K - 1; ++j) store<T, VEC>(p.fin, ((long long)s * (K - 1) + K - 2 - j) * p.D + d, hist[j]);
    }
  }
}

template <typename T, int K, int VEC, bool SEQ>
__global__ void __launch_bounds__(kWarps * 32) conv_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int U = VEC >= 4 ? 4 : 8;
  __shared__ float red[kWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = (p.D / VEC + 31) / 32;
  const long long blk = blockIdx.x / groups;
  const int d0 = (int)(blockIdx.x - blk * groups) * 32 * VEC;
  int d = d0 + lane * VEC;
  const At a = run_of(p, blk * kWarps + warp);
  const bool on = d < p.D;
  if (!on) d = 0;
  Vals<VEC> dw[K + 1];  // the taps' gradients, then the bias's
#pragma unroll
  for (int k = 0; k <= K; ++k) dw[k] = zeros<VEC>();
  if (a.on) {
    const Taps<K, VEC> taps(p, d);
    const T* x = static_cast<const T*>(p.x) + a.row * p.x_b + d;
    const T* dy = static_cast<const T*>(p.dy) + (long long)a.row * p.L * p.D + d;
    T* dx = static_cast<T*>(p.dx) + (long long)a.row * p.L * p.D + d;
    Vals<VEC> hist[K - 1], acc[K];  // acc[j]: the gradient of the row j before
    int first = rows_before<T, K, VEC, SEQ>(p, x, a.t0, d, hist);  // the sequence's first token, or any earlier place
#pragma unroll
    for (int j = 0; j < K; ++j) acc[j] = zeros<VEC>();
    const int stop = min(p.L, a.t1 + K - 1);
    // the token's gradient of p; `own`: its products are this run's
    const auto token = [&](const Vals<VEC>& v, const Vals<VEC>& gy, bool own, bool none) {
      Vals<VEC> g = gy;
      if (p.act) {
        const Vals<VEC> q = taps.at(v, hist);
#pragma unroll
        for (int j = 0; j < Vals<VEC>::H; ++j) {  // silu'(q) = s (1 + q (1 - s))
          const float2 sg = sigmoid2(q.v[j]), one = make_float2(1.f, 1.f);
          const float2 rest = __fadd2_rn(one, make_float2(-sg.x, -sg.y));
          g.v[j] = __fmul2_rn(g.v[j], __fmul2_rn(sg, __ffma2_rn(q.v[j], rest, one)));
        }
      }
      if (none) g = zeros<VEC>();  // a token of no sequence
#pragma unroll
      for (int j = 0; j < K; ++j) acc[j] = fma_of(taps.w[K - 1 - j], g, acc[j]);
      if (own && !none) {
        dw[K - 1] = fma_of(g, v, dw[K - 1]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) dw[K - 2 - j] = fma_of(g, hist[j], dw[K - 2 - j]);
#pragma unroll
        for (int j = 0; j < Vals<VEC>::H; ++j) dw[K].v[j] = __fadd2_rn(dw[K].v[j], g.v[j]);
      }
    };
    const auto shift = [&](const Vals<VEC>& v) {
#pragma unroll
      for (int j = K - 1; j > 0; --j) acc[j] = acc[j - 1];
      acc[0] = zeros<VEC>();
      push<K, VEC>(hist, v);
    };
    // row tok of the sequence (before `first`: of its initial state) has its whole gradient
    const auto emit = [&](int tok, int s, const Vals<VEC>& g) {
      if (tok >= first) {
        if (on && tok >= a.t0 && tok < a.t1) store<T, VEC>(dx, (long long)tok * p.D, g);
      } else if (on && p.dinit && s >= 0 && first >= a.t0) {
        store<T, VEC>(p.dinit, ((long long)s * (K - 1) + K - 1 + tok - first) * p.D + d, g);
      }
    };
    bool done = false;
    for (int t = a.t0; t < stop && !done;) {
      // past the rows before the run, before its end, within a sequence
      if (t >= max(a.t0, first) + K - 1 && t + U <= a.t1 && plain<U, SEQ>(p, t)) {
        Pack<T, VEC> in[U], gy[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
          in[i] = load<T, VEC>(x, (t + i) * p.x_l), gy[i] = load<T, VEC>(dy, (long long)(t + i) * p.D);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const Vals<VEC> v = unpack<T, VEC>(in[i]);
          token(v, unpack<T, VEC>(gy[i]), true, false);
          if (on) store<T, VEC>(dx, (long long)(t + i - (K - 1)) * p.D, acc[K - 1]);
          shift(v);
        }
        t += U;
        continue;
      }
      for (const int end = min(t + U, stop); t < end; ++t) {
        const int s = SEQ ? p.seq[t] : a.row;
        if (starts<SEQ>(p, t)) {
          if (t >= a.t1) {
            done = true;
            break;
          }
          initial_rows<T, K, VEC>(p, s, d, hist);
          first = t;
#pragma unroll
          for (int j = 0; j < K; ++j) acc[j] = zeros<VEC>();
        }
        const Vals<VEC> v = unpack<T, VEC>(load<T, VEC>(x, t * p.x_l));
        token(v, unpack<T, VEC>(load<T, VEC>(dy, (long long)t * p.D)), t < a.t1, s < 0);
        emit(t - (K - 1), s, acc[K - 1]);
        if (ends<SEQ>(p, t)) {
#pragma unroll
          for (int j = K - 2; j >= 0; --j) {
            if (p.dfin && s >= 0) {
              const Vals<VEC> f = unpack<T, VEC>(load<T, VEC>(p.dfin, ((long long)s * (K - 1) + K - 2 - j) * p.D + d));
#pragma unroll
              for (int e = 0; e < Vals<VEC>::H; ++e) acc[j].v[e] = __fadd2_rn(acc[j].v[e], f.v[e]);
            }
            emit(t - j, s, acc[j]);
          }
        }
        shift(v);
      }
    }
  }
  // the block's runs together, a tap at a time
  float* part = p.part + blk * p.D * (K + 1);
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[warp][lane * VEC + e] = e % 2 ? dw[k].v[e / 2].y : dw[k].v[e / 2].x;
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * VEC; c += kWarps * 32) {
      if (d0 + c < p.D) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) v += red[q][c];
        part[k < K ? (long long)(d0 + c) * K + k : (long long)p.D * K + d0 + c] = v;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------ single token
struct StepParams {
  int rows, D, act, slots;
  long long x_b, state_b;
  const void* x;
  const float *w, *b;
  const int* index;
  void *state, *y;  // [slots, K - 1, D], [rows, D]
};

template <typename T, int K>
__global__ void __launch_bounds__(128) conv_step_kernel(const __grid_constant__ StepParams p) {
  const int tiles = (p.D + 127) / 128, row = blockIdx.x / tiles, d = (blockIdx.x - row * tiles) * 128 + threadIdx.x;
  const int ok = scan::slot_state(p.index, row, p.slots);
  if (d >= p.D) return;
  T* y = static_cast<T*>(p.y) + (long long)row * p.D + d;
  if (ok <= 0) {
    *y = from_f<T>(ok < 0 ? __int_as_float(0x7fffffff) : 0.f);
    return;
  }
  T* state = static_cast<T*>(p.state) + (long long)(p.index ? p.index[row] : row) * p.state_b + d;
  const T x = static_cast<const T*>(p.x)[row * p.x_b + d];
  T old[K - 1];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) old[k] = state[(long long)k * p.D];
  float q = fmaf(p.w[(long long)d * K + K - 1], to_f(x), p.b ? p.b[d] : 0.f);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) q = fmaf(p.w[(long long)d * K + k], to_f(old[k]), q);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) state[(long long)k * p.D] = k + 1 < K - 1 ? old[k + 1] : x;
  *y = from_f<T>(p.act ? q * scan::sigmoid(q) : q);
}

// ------------------------------------------------------------------------------ host
static int check(const char* who, int rows, int L, int D, int K, int act, int dt) {
  TTT_REQUIRE(rows >= 1 && L >= 1 && D >= 1, TTT_ERR_SHAPE, "%s: sizes must be positive, got rows=%d L=%d D=%d", who,
              rows, L, D);
  TTT_REQUIRE(K >= 2 && K <= 4, TTT_ERR_SHAPE, "%s: %d taps, 2 to 4 are supported", who, K);
  TTT_REQUIRE((long long)rows * L < (1LL << 31) - 4096, TTT_ERR_SHAPE, "%s: %lld tokens are too many", who,
              (long long)rows * L);
  TTT_REQUIRE(act == 0 || act == 1, TTT_ERR_SHAPE, "%s: bad activation code %d", who, act);
  TTT_REQUIRE(valid_dtype(dt), TTT_ERR_DTYPE, "%s: bad dtype code %d", who, dt);
  return TTT_OK;
}

// Tokens of a run: short enough that the device has work for 16 warps an SM, at least 16
// (the K - 1 rows before a run are read again for it).
static int run_tokens(int rows, int L, int D, int vec) {
  const long long want = (long long)scan::sm_count() * 16, warps = (long long)rows * ((D / vec + 31) / 32);
  int run = 128;
  while (run > 16 && warps * ((L + run - 1) / run) < want) run >>= 1;
  return run;
}

static bool vectors(int D, int vec, int elem, const long long* strides, std::initializer_list<const void*> ptrs) {
  if (D % vec || strides[0] % vec || strides[1] % vec) return false;
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % (vec * elem)) return false;
  return true;
}

static void split(Params& p, int vec) {
  p.run = run_tokens(p.rows, p.L, p.D, vec);
  p.runs = (p.L + p.run - 1) / p.run;
}
static long long run_blocks(const Params& p) { return ((long long)p.rows * p.runs + kWarps - 1) / kWarps; }

template <typename T, int K, int VEC, bool BWD>
static int launch(const Params& p, cudaStream_t st, const char* who) {
  const long long grid = run_blocks(p) * ((p.D / VEC + 31) / 32);
  TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
  const auto kernel = [&] {
    if constexpr (BWD) return p.seq ? conv_bwd_kernel<T, K, VEC, true> : conv_bwd_kernel<T, K, VEC, false>;
    else return p.seq ? conv_fwd_kernel<T, K, VEC, true> : conv_fwd_kernel<T, K, VEC, false>;
  }();
  kernel<<<(unsigned)grid, kWarps * 32, 0, st>>>(p);
  return check_launch(who);
}
template <typename T, int VEC, bool BWD>
static int launch_k(const Params& p, int K, cudaStream_t st, const char* who) {
  return K == 2 ? launch<T, 2, VEC, BWD>(p, st, who)
         : K == 3 ? launch<T, 3, VEC, BWD>(p, st, who)
                  : launch<T, 4, VEC, BWD>(p, st, who);
}
template <int VEC16, int VEC32, bool BWD>
static int launch_t(const Params& p, int K, int dt, bool vec, cudaStream_t st, const char* who) {
  if (dt == DT_BF16)
    return vec ? launch_k<__nv_bfloat16, VEC16, BWD>(p, K, st, who) : launch_k<__nv_bfloat16, 1, BWD>(p, K, st, who);
  if (dt == DT_F16) return vec ? launch_k<__half, VEC16, BWD>(p, K, st, who) : launch_k<__half, 1, BWD>(p, K, st, who);
  return vec ? launch_k<float, VEC32, BWD>(p, K, st, who) : launch_k<float, 1, BWD>(p, K, st, who);
}

}  // namespace conv
}  // namespace ttt

using namespace ttt;

extern "C" int ttt_causal_conv_fwd(int rows, int L, int D, int K, const void* x, int dt, const long long* strides,
                                   const float* w, const float* b, int act, const int* seq, const void* init,
                                   void* fin, void* y, void* stream) {
  const char* who = "ttt_causal_conv_fwd";
  int rc = conv::check(who, rows, L, D, K, act, dt);
  if (rc) return rc;
  TTT_REQUIRE(x && w && y && strides, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(!seq || rows == 1, TTT_ERR_SHAPE, "%s: packed sequences lie in one row, got %d", who, rows);
  conv::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.act = act, p.x = x, p.x_b = strides[0], p.x_l = strides[1];
  p.w = w, p.b = b, p.seq = seq, p.init = init, p.fin = fin, p.y = y;
  const int elem = dt == DT_F32 ? 4 : 2;
  const bool on = conv::vectors(D, 4, elem, strides, {x, init, fin, y});
  conv::split(p, on ? 4 : 1);
  return conv::launch_t<4, 4, false>(p, K, dt, on, static_cast<cudaStream_t>(stream), who);
}

// The backward holds K rows of x, of gradients and of weight sums per channel: 8-byte vectors.
static size_t conv_bwd_need(conv::Params& p, int K, int dt, bool vec) {
  conv::split(p, vec ? (dt == DT_F32 ? 2 : 4) : 1);
  return (size_t)conv::run_blocks(p) * p.D * (K + 1) * sizeof(float);
}

extern "C" size_t ttt_causal_conv_bwd_scratch_bytes(int rows, int L, int D, int K, int dt) {
  if (conv::check("ttt_causal_conv_bwd_scratch_bytes", rows, L, D, K, 0, dt)) return 0;
  conv::Params p{};
  p.rows = rows, p.L = L, p.D = D;
  const size_t a = conv_bwd_need(p, K, dt, false), b = conv_bwd_need(p, K, dt, true);
  return a > b ? a : b;  // the strides and addresses choose between the two
}

extern "C" int ttt_causal_conv_bwd(int rows, int L, int D, int K, const void* x, int dt, const long long* strides,
                                   const float* w, const float* b, int act, const int* seq, const void* init,
                                   const void* dy, const void* dfin, void* dx, void* dinit, float* dparams,
                                   void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "ttt_causal_conv_bwd";
  int rc = conv::check(who, rows, L, D, K, act, dt);
  if (rc) return rc;
  TTT_REQUIRE(x && w && dy && dx && dparams && strides, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(!seq || rows == 1, TTT_ERR_SHAPE, "%s: packed sequences lie in one row, got %d", who, rows);
  conv::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.act = act, p.x = x, p.x_b = strides[0], p.x_l = strides[1];
  p.w = w, p.b = b, p.seq = seq, p.init = init, p.dy = dy, p.dfin = dfin, p.dx = dx, p.dinit = dinit;
  const int elem = dt == DT_F32 ? 4 : 2;
  const bool on = conv::vectors(D, 8 / elem, elem, strides, {x, init, dy, dfin, dx, dinit});
  const size_t need = conv_bwd_need(p, K, dt, on);
  TTT_REQUIRE(scratch && scratch_bytes >= need, TTT_ERR_SCRATCH, "%s: scratch of %zu bytes needed, got %zu", who, need,
              scratch ? scratch_bytes : (size_t)0);
  p.part = static_cast<float*>(scratch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = conv::launch_t<4, 2, true>(p, K, dt, on, st, who))) return rc;
  return scan::column_sum(p.part, conv::run_blocks(p), (long long)D * (K + 1), dparams, st, who);
}

extern "C" int ttt_causal_conv_step(int rows, int D, int K, int slots, const void* x, int dt, const long long* strides,
                                    const float* w, const float* b, int act, const int* index, void* state, void* y,
                                    void* stream) {
  const char* who = "ttt_causal_conv_step";
  int rc = conv::check(who, rows, 1, D, K, act, dt);
  if (rc) return rc;
  TTT_REQUIRE(x && w && state && y && strides, TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(slots >= 1 && (index || slots >= rows), TTT_ERR_SHAPE, "%s: %d states for %d rows", who, slots, rows);
  const long long grid = (long long)rows * ((D + 127) / 128);
  TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
  conv::StepParams p{};
  p.rows = rows, p.D = D, p.act = act, p.slots = slots, p.x_b = strides[0], p.state_b = strides[1];
  p.x = x, p.w = w, p.b = b, p.index = index, p.state = state, p.y = y;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    if (K == 2) conv::conv_step_kernel<T, 2><<<(unsigned)grid, 128, 0, st>>>(p);
    else if (K == 3) conv::conv_step_kernel<T, 3><<<(unsigned)grid, 128, 0, st>>>(p);
    else conv::conv_step_kernel<T, 4><<<(unsigned)grid, 128, 0, st>>>(p);
    return check_launch(who);
  };
  return dt == DT_BF16 ? go(__nv_bfloat16{}) : dt == DT_F16 ? go(__half{}) : go(float{});
}
