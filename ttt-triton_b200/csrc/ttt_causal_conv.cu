// Short causal convolution along the sequence, per channel, with K = 2 .. 4 taps:
//
//   p[t] = bias + sum_k w[k] x[t - K + 1 + k],  y = p or p sigmoid(p)
//
// Rows before a sequence's first token are its initial state's K - 1 rows, or zero; the final
// state is its last K - 1 rows. It moves every value once in and once out with a handful of
// operations each, so memory bounds it: a thread holds VEC adjacent channels (a vector load
// per token), walks a run of tokens with the last K - 1 rows in registers, and loads several
// tokens ahead; a warp covers 32 adjacent vectors of one run, a block 8 runs.
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
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> zero_pack() {
  Pack<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = from_f<T>(0.f);
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load(const void* base, long long at) {
  return *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(base) + at);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(void* base, long long at, const float (&x)[VEC]) {
  Pack<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = from_f<T>(x[e]);
  *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(base) + at) = r;
}

// The channels' weights, tap 0 on the oldest row.
template <int K, int VEC>
struct Taps {
  float w[K][VEC], b[VEC];
  __device__ __forceinline__ Taps(const Params& p, int d, bool on) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][e] = on ? p.w[(long long)(d + e) * K + k] : 0.f;
      b[e] = on && p.b ? p.b[d + e] : 0.f;
    }
  }
};

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
__device__ __forceinline__ bool starts(const Params& p, int t) { return p.seq ? scan::seq_starts(p.seq, t) : t == 0; }
__device__ __forceinline__ bool ends(const Params& p, int t) {
  return p.seq ? scan::seq_ends(p.seq, t, p.L) : t == p.L - 1;
}

// The K - 1 rows before a sequence's first token: hist[0] is the nearest.
template <typename T, int K, int VEC>
__device__ __forceinline__ void initial_rows(const Params& p, int s, int d, float (&hist)[K - 1][VEC]) {
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    Pack<T, VEC> r = zero_pack<T, VEC>();
    if (p.init && s >= 0) r = load<T, VEC>(p.init, ((long long)s * (K - 1) + K - 2 - j) * p.D + d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) hist[j][e] = to_f(r.v[e]);
  }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kWarps * 32) conv_fwd_kernel(const __grid_constant__ Params p) {
  constexpr int U = 8;  // tokens loaded together
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = (p.D / VEC + 31) / 32;
  const long long blk = blockIdx.x / groups;
  const int d = ((int)(blockIdx.x - blk * groups) * 32 + lane) * VEC;
  const At a = run_of(p, blk * kWarps + warp);
  if (!a.on || d >= p.D) return;
  const Taps<K, VEC> taps(p, d, true);
  const T* x = static_cast<const T*>(p.x) + a.row * p.x_b + d;
  float hist[K - 1][VEC] = {};
  for (int t = max(0, a.t0 - (K - 1)); t < a.t1;) {
    const int n = min(U, (t < a.t0 ? a.t0 : a.t1) - t);
    Pack<T, VEC> in[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i < n) in[i] = load<T, VEC>(x, (t + i) * p.x_l);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= n) break;
      const int tok = t + i, s = p.seq ? p.seq[tok] : a.row;
      if (starts(p, tok)) initial_rows<T, K, VEC>(p, s, d, hist);
      float v[VEC], y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] = to_f(in[i].v[e]);
        float q = fmaf(taps.w[K - 1][e], v[e], taps.b[e]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) q = fmaf(taps.w[K - 2 - j][e], hist[j][e], q);
        y[e] = s < 0 ? 0.f : p.act ? q * scan::sigmoid(q) : q;
#pragma unroll
        for (int j = K - 2; j > 0; --j) hist[j][e] = hist[j - 1][e];
        hist[0][e] = v[e];
      }
      if (tok >= a.t0) {
        store<T, VEC>(p.y, ((long long)a.row * p.L + tok) * p.D + d, y);
        if (p.fin && s >= 0 && ends(p, tok))
#pragma unroll
          for (int j = 0; j < K - 1; ++j)
            store<T, VEC>(p.fin, ((long long)s * (K - 1) + K - 2 - j) * p.D + d, hist[j]);
      }
    }
    t += n;
  }
}

template <typename T, int K, int VEC>
__global__ void __launch_bounds__(kWarps * 32) conv_bwd_kernel(const __grid_constant__ Params p) {
  __shared__ float red[kWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = (p.D / VEC + 31) / 32;
  const long long blk = blockIdx.x / groups;
  const int d0 = (int)(blockIdx.x - blk * groups) * 32 * VEC, d = d0 + lane * VEC;
  const At a = run_of(p, blk * kWarps + warp);
  float dw[K + 1][VEC] = {};  // the taps' gradients, then the bias's
  if (a.on && d < p.D) {
    const Taps<K, VEC> taps(p, d, true);
    const T* x = static_cast<const T*>(p.x) + a.row * p.x_b + d;
    const T* dy = static_cast<const T*>(p.dy) + (long long)a.row * p.L * p.D + d;
    T* dx = static_cast<T*>(p.dx) + (long long)a.row * p.L * p.D + d;
    float hist[K - 1][VEC] = {}, acc[K][VEC] = {};  // acc[j]: the gradient of the row j before
    int first = -K;  // the sequence's first token, or any earlier place
    const int stop = min(p.L, a.t1 + K - 1);
    // row tok of the sequence (before `first`: of its initial state) has its whole gradient
    const auto emit = [&](int tok, int s, const float (&g)[VEC]) {
      if (tok >= first) {
        if (tok >= a.t0 && tok < a.t1) store<T, VEC>(dx, (long long)tok * p.D, g);
      } else if (p.dinit && s >= 0 && first >= a.t0) {
        store<T, VEC>(p.dinit, ((long long)s * (K - 1) + K - 1 + tok - first) * p.D + d, g);
      }
    };
    for (int tok = max(0, a.t0 - (K - 1)); tok < stop; ++tok) {
      const int s = p.seq ? p.seq[tok] : a.row;
      if (starts(p, tok)) {
        if (tok >= a.t1) break;
        initial_rows<T, K, VEC>(p, s, d, hist);
        first = tok;
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[j][e] = 0.f;
      }
      const Pack<T, VEC> in = load<T, VEC>(x, tok * p.x_l);
      float v[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = to_f(in.v[e]);
      if (tok >= a.t0) {
        const Pack<T, VEC> gy = load<T, VEC>(dy, (long long)tok * p.D);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float q = fmaf(taps.w[K - 1][e], v[e], taps.b[e]);
#pragma unroll
          for (int j = 0; j < K - 1; ++j) q = fmaf(taps.w[K - 2 - j][e], hist[j][e], q);
          float g = to_f(gy.v[e]);
          if (p.act) g *= scan::silu_grad(q, scan::sigmoid(q));
          if (s < 0) g = 0.f;  // a token of no sequence
#pragma unroll
          for (int j = 0; j < K; ++j) acc[j][e] = fmaf(taps.w[K - 1 - j][e], g, acc[j][e]);
          if (tok < a.t1 && s >= 0) {
            dw[K - 1][e] = fmaf(g, v[e], dw[K - 1][e]);
#pragma unroll
            for (int j = 0; j < K - 1; ++j) dw[K - 2 - j][e] = fmaf(g, hist[j][e], dw[K - 2 - j][e]);
            dw[K][e] += g;
          }
        }
        emit(tok - (K - 1), s, acc[K - 1]);
        if (ends(p, tok)) {
#pragma unroll
          for (int j = K - 2; j >= 0; --j) {
            if (p.dfin && s >= 0) {
              const Pack<T, VEC> f = load<T, VEC>(p.dfin, ((long long)s * (K - 1) + K - 2 - j) * p.D + d);
#pragma unroll
              for (int e = 0; e < VEC; ++e) acc[j][e] += to_f(f.v[e]);
            }
            emit(tok - j, s, acc[j]);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
#pragma unroll
        for (int j = K - 1; j > 0; --j) acc[j][e] = acc[j - 1][e];
        acc[0][e] = 0.f;
#pragma unroll
        for (int j = K - 2; j > 0; --j) hist[j][e] = hist[j - 1][e];
        hist[0][e] = v[e];
      }
    }
  }
  // the block's runs together, a tap at a time
  float* part = p.part + blk * p.D * (K + 1);
#pragma unroll
  for (int k = 0; k <= K; ++k) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[warp][lane * VEC + e] = dw[k][e];
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
  if (BWD) conv_bwd_kernel<T, K, VEC><<<(unsigned)grid, kWarps * 32, 0, st>>>(p);
  else conv_fwd_kernel<T, K, VEC><<<(unsigned)grid, kWarps * 32, 0, st>>>(p);
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
  const int elem = dt == DT_F32 ? 4 : 2, vec = 16 / elem;
  const bool on = conv::vectors(D, vec, elem, strides, {x, init, fin, y});
  conv::split(p, on ? vec : 1);
  return conv::launch_t<8, 4, false>(p, K, dt, on, static_cast<cudaStream_t>(stream), who);
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
