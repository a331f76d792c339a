// Selective state space scan, backward (the recurrence is in selective_scan.cuh):
//
//   dy = dout silu(z),  g[t] = C dy + a[t+1] g[t+1],  q = g a h[t-1]
//   dC = sum_d h dy,  dB = sum_d g dt u,  s1 = <g, B>,  s2 = <q, A>
//   du = dt s1 + D dy,  ddt = u s1 + s2,  dA = sum q dt,  dz = dout y silu'(z)
//
// A CTA walks its channels' time axis backwards in tiles of TB tokens, each starting at a
// state that the forward kept. The tile's states are run forward again, SUB tokens at a time
// held in registers (decays a and a h[t-1]), then g runs back through them. Sums over a
// channel's states (s1, s2 and y) go through shared memory, those over channels (dB, dC)
// through shuffles within a warp and shared memory between warps; what the CTAs of a group
// have of dB and dC, and what the rows and pieces have of dA, dD and dbias, is written as
// partials and added in a fixed order afterwards, so that results do not depend on timing.
#include "selective_scan.cuh"

namespace ttt {
namespace scan {

template <int LN, int NPT>
struct Bwd {
  static constexpr int THREADS = 256, WARPS = THREADS / 32;
  static constexpr int DT = THREADS / LN;     // channels of a CTA
  static constexpr int NP = LN * NPT;         // states, padded
  static constexpr int TB = 64 / NPT;         // tokens of a tile: save_every()
  static constexpr int SUB = TB / 2;          // tokens whose states are in registers
  static constexpr int PAIRS = TB * DT / THREADS > 0 ? TB * DT / THREADS : 1;
  struct Smem {
    float B[TB * NP], C[TB * NP];
    float dt[TB * DT], dtu[TB * DT], dy[TB * DT];
    float s1[TB * THREADS], s2[TB * THREADS], s3[TB * THREADS];
    float dB[WARPS][TB * NP], dC[WARPS][TB * NP];
    float red[THREADS];
    SeqMask m;
  };
};

template <typename T, int LN, int NPT>
__global__ void __launch_bounds__(256) scan_bwd_kernel(const __grid_constant__ Params p) {
  using F = Bwd<LN, NPT>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // lane -> channel and states: the low two bits and those above the LN state threads' are
  // the channel's
  const int nl = (lane >> 2) % LN, cl = warp * (32 / LN) + (lane & 3) + 4 * ((lane >> 2) / LN);
  const int n0 = nl * NPT, at = cl * LN + nl;
  const int d = w.g * p.Dg + w.d0 + cl;
  const bool on = w.d0 + cl < p.Dg;
  const int pc = tid % F::DT, pd = w.g * p.Dg + w.d0 + pc;  // channel in the element-wise passes
  const bool pon = w.d0 + pc < p.Dg;
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const long long DN = (long long)p.D * p.N;

  float A2[NPT], carry[NPT], dA[NPT];
  load_states<NPT>(p.A, d, n0, p.N, on, A2);
#pragma unroll
  for (int i = 0; i < NPT; ++i) A2[i] *= kLog2e, dA[i] = 0.f;
  if (p.nchunks > 1)
    load_states<NPT>(p.cstate + ((long long)w.row * p.nchunks + w.piece) * DN, d, n0, p.N, on, carry);
  else
    load_states<NPT>(p.dfin + w.row * DN, d, n0, p.N, on && p.dfin && !p.seq, carry);
  const float skip = pon && p.Dskip ? p.Dskip[pd] : 0.f, bias = pon && p.bias ? p.bias[pd] : 0.f;
  const T* u = static_cast<const T*>(p.u) + w.row * p.u_b + pd;
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + pd;
  const T* z = p.z ? static_cast<const T*>(p.z) + w.row * p.z_b + pd : nullptr;
  const T* B = static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const T* C = static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g;
  const long long row0 = (long long)w.row * p.L;
  float sum_D = 0.f, sum_bias = 0.f;

  for (int tile = (tend - 1) / F::TB; tile >= tbeg / F::TB; --tile) {
    const int t0 = tile * F::TB;
    float uu[F::PAIRS], raw[F::PAIRS], zz[F::PAIRS], dd[F::PAIRS];
    if (p.seq) stage_masks<F::TB>(&s.m, p.seq, t0, tend, p.L);
#pragma unroll
    for (int k = 0; k < F::PAIRS; ++k) {
      const int t = tid / F::DT + k * LN, tok = t0 + t;
      float dt = 0.f, dy = 0.f;
      uu[k] = raw[k] = zz[k] = dd[k] = 0.f;
      if (t < F::TB) {
        if (pon && tok < tend && !(p.seq && p.seq[tok] < 0)) {
          uu[k] = to_f(u[tok * p.u_l]);
          raw[k] = to_f(delta[tok * p.delta_l]) + bias;
          dt = step_size(p, raw[k]);
          dd[k] = dy = to_f(static_cast<const T*>(p.dout)[(row0 + tok) * p.D + pd]);
          if (z) {
            zz[k] = to_f(z[tok * p.z_l]);
            dy *= zz[k] * sigmoid(zz[k]);
          }
        }
        s.dt[t * F::DT + pc] = dt, s.dtu[t * F::DT + pc] = dt * uu[k], s.dy[t * F::DT + pc] = dy;
      }
    }
    stage_rows<T, F::NP, F::TB, F::THREADS>(s.B, B, p.B_l, t0, tend, p.N, p.seq, p.quads);
    stage_rows<T, F::NP, F::TB, F::THREADS>(s.C, C, p.C_l, t0, tend, p.N, p.seq, p.quads);
    __syncthreads();

    float h0[NPT], hm[NPT];  // the states before the tile's first token and before its second half
    load_states<NPT>(p.hsave + ((long long)w.row * p.nsave + tile) * DN, d, n0, p.N, on, h0);
    const auto restart = [&](int t, float (&h)[NPT]) {
      if (p.seq && (s.m.start >> t & 1)) {
        const int q = p.seq[t0 + t];
        load_states<NPT>(p.init + q * DN, d, n0, p.N, on && q >= 0 && p.init, h);
      }
    };
#pragma unroll
    for (int i = 0; i < NPT; ++i) hm[i] = h0[i];
#pragma unroll
    for (int t = 0; t < F::SUB; ++t) {
      restart(t, hm);
      const float dt = s.dt[t * F::DT + cl], dtu = s.dtu[t * F::DT + cl];
#pragma unroll
      for (int i = 0; i < NPT; ++i)
        hm[i] = fmaf(ex2(dt * A2[i]), hm[i], dtu * s.B[t * F::NP + n0 + i]);
    }
#pragma unroll 1
    for (int half = 1; half >= 0; --half) {
      const int b = half * F::SUB;
      float a[F::SUB][NPT], ah[F::SUB][NPT], h[NPT];
#pragma unroll
      for (int i = 0; i < NPT; ++i) h[i] = half ? hm[i] : h0[i];
#pragma unroll
      for (int k = 0; k < F::SUB; ++k) {
        const int t = b + k;
        restart(t, h);
        const float dt = s.dt[t * F::DT + cl], dtu = s.dtu[t * F::DT + cl];
#pragma unroll
        for (int i = 0; i < NPT; ++i) {
          a[k][i] = ex2(dt * A2[i]);
          ah[k][i] = a[k][i] * h[i];
          h[i] = fmaf(dtu, s.B[t * F::NP + n0 + i], ah[k][i]);
        }
      }
#pragma unroll
      for (int k = F::SUB - 1; k >= 0; --k) {
        const int t = b + k;
        const float dt = s.dt[t * F::DT + cl], dtu = s.dtu[t * F::DT + cl], dy = s.dy[t * F::DT + cl];
        if (p.seq && (s.m.end >> t & 1)) {
          const int q = p.seq[t0 + t];
          load_states<NPT>(p.dfin + q * DN, d, n0, p.N, on && q >= 0 && p.dfin, carry);
        }
        float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int i = 0; i < NPT; ++i) {
          const float Bn = s.B[t * F::NP + n0 + i], Cn = s.C[t * F::NP + n0 + i];
          const float g = fmaf(Cn, dy, carry[i]), hn = fmaf(dtu, Bn, ah[k][i]), q = g * ah[k][i];
          s1 = fmaf(g, Bn, s1), s2 = fmaf(q, A2[i], s2), s3 = fmaf(hn, Cn, s3);
          dA[i] = fmaf(q, dt, dA[i]);
          carry[i] = a[k][i] * g;
          float vb = g * dtu, vc = hn * dy;  // summed over the warp's channels
#pragma unroll
          for (int o = 1; o < 32; o <<= 1)
            if (o < 4 || o >= 4 * LN)
              vb += __shfl_xor_sync(0xffffffffu, vb, o), vc += __shfl_xor_sync(0xffffffffu, vc, o);
          if ((lane & 3) == 0 && (lane >> 2) < LN)
            s.dB[warp][t * F::NP + n0 + i] = vb, s.dC[warp][t * F::NP + n0 + i] = vc;
        }
        s.s1[t * F::THREADS + at] = s1, s.s2[t * F::THREADS + at] = s2, s.s3[t * F::THREADS + at] = s3;
        if (p.seq && (s.m.start >> t & 1)) {
          const int q = p.seq[t0 + t];
          if (p.dinit) store_states<NPT>(p.dinit + q * DN, d, n0, p.N, on && q >= 0, carry);
        }
      }
    }
    __syncthreads();

#pragma unroll
    for (int k = 0; k < F::PAIRS; ++k) {
      const int t = tid / F::DT + k * LN, tok = t0 + t;
      if (t < F::TB && pon && tok < tend) {
        float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int j = 0; j < LN; ++j) {
          const int e = t * F::THREADS + pc * LN + j;
          s1 += s.s1[e], s2 += s.s2[e], s3 += s.s3[e];
        }
        const float dt = s.dt[t * F::DT + pc], dy = s.dy[t * F::DT + pc];
        float du = fmaf(dt, s1, skip * dy), ddt = fmaf(uu[k], s1, s2 * kLn2), dz = 0.f;
        if (p.softplus) ddt *= sigmoid(raw[k]);
        if (z) dz = dd[k] * fmaf(skip, uu[k], s3) * silu_grad(zz[k], sigmoid(zz[k]));
        if (p.seq && !(s.m.in >> t & 1)) du = ddt = dz = 0.f;  // a token of no sequence
        else sum_D = fmaf(uu[k], dy, sum_D), sum_bias += ddt;
        const long long o = (row0 + tok) * p.D + pd;
        static_cast<T*>(p.du)[o] = from_f<T>(du);
        static_cast<T*>(p.ddelta)[o] = from_f<T>(ddt);
        if (z) static_cast<T*>(p.dz)[o] = from_f<T>(dz);
      }
    }
    const int tile_g = w.d0 / F::DT;
    for (int i = tid; i < F::TB * F::NP; i += F::THREADS) {
      const int t = i / F::NP, n = i - t * F::NP;
      if (t0 + t < tend && n < p.N) {
        float vb = 0.f, vc = 0.f;
#pragma unroll
        for (int k = 0; k < F::WARPS; ++k) vb += s.dB[k][i], vc += s.dC[k][i];
        const bool out = p.seq && !(s.m.in >> t & 1);
        const long long o = (((long long)tile_g * p.rows * p.L + row0 + t0 + t) * p.G + w.g) * p.N + n;
        p.part_B[o] = out ? 0.f : vb, p.part_C[o] = out ? 0.f : vc;
      }
    }
    __syncthreads();
  }

  if (p.dinit && !p.seq && tbeg == 0) store_states<NPT>(p.dinit + w.row * DN, d, n0, p.N, on, carry);
  float* part = p.part_p + ((long long)w.row * p.nchunks + w.piece) * p.D * (p.N + 2);
  store_states<NPT>(part, d, n0, p.N, on, dA);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    s.red[tid] = k ? sum_bias : sum_D;
    __syncthreads();
    if (tid < F::DT && pon) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < LN; ++j) v += s.red[tid + j * F::DT];
      part[DN + (long long)k * p.D + pd] = v;
    }
    __syncthreads();
  }
}

// dB, dC from the channel tiles' partials, in one order.
template <typename T>
__global__ void __launch_bounds__(256) scan_sum_tiles_kernel(const float* part_B, const float* part_C, int tiles,
                                                             long long n, T* dB, T* dC) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float b = 0.f, c = 0.f;
  for (int k = 0; k < tiles; ++k) b += part_B[k * n + i], c += part_C[k * n + i];
  dB[i] = from_f<T>(b), dC[i] = from_f<T>(c);
}

// 32 columns, 16 groups of rows.
__global__ void __launch_bounds__(512) column_sum_kernel(const float* part, long long M, long long W, float* out) {
  __shared__ float red[16][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  const long long w = (long long)blockIdx.x * 32 + c;
  float v = 0.f;
  if (w < W)
    for (long long m = r; m < M; m += 16) v += part[m * W + w];
  red[r][c] = v;
  __syncthreads();
  if (r == 0 && w < W) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += red[k][c];
    out[w] = v;
  }
}
int column_sum(const float* part, long long M, long long W, float* out, cudaStream_t st, const char* who) {
  const long long grid = (W + 31) / 32;
  TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld columns are too many", who, W);
  column_sum_kernel<<<(unsigned)grid, 512, 0, st>>>(part, M, W, out);
  return check_launch(who);
}

// ------------------------------------------------------------------------------ host
static int channels_of_a_cta(int N) { return 256 / shape_of(N).LN; }

struct BwdScratch {
  size_t tiles, part_bc, part_p, states;  // bytes but for tiles
};
static BwdScratch bwd_scratch(int rows, int L, int D, int G, int N, int nchunks) {
  BwdScratch s;
  s.tiles = (D / G + channels_of_a_cta(N) - 1) / channels_of_a_cta(N);
  s.part_bc = s.tiles * rows * L * G * N * sizeof(float);
  s.part_p = (size_t)rows * nchunks * D * (N + 2) * sizeof(float);
  return s;
}

template <typename T>
static int launch_bwd(Params p, void* dB, void* dC, float* dparams, cudaStream_t st, const char* who) {
  int rc = dispatch(p.N, [&](auto ln, auto npt) {
    using F = Bwd<decltype(ln)::value, decltype(npt)::value>;
    auto kernel = scan_bwd_kernel<T, decltype(ln)::value, decltype(npt)::value>;
    const int rc2 = prepare_smem(kernel, sizeof(typename F::Smem), who);
    if (rc2) return rc2;
    const long long grid = (long long)p.tiles * p.G * p.nchunks * p.rows;
    TTT_REQUIRE(grid < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld blocks are too many", who, grid);
    kernel<<<(unsigned)grid, F::THREADS, sizeof(typename F::Smem), st>>>(p);
    return check_launch(who);
  });
  if (rc) return rc;
  const long long n = (long long)p.rows * p.L * p.G * p.N;
  TTT_REQUIRE((n + 255) / 256 < (1LL << 31), TTT_ERR_SHAPE, "%s: %lld values of dB are too many", who, n);
  scan_sum_tiles_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p.part_B, p.part_C, p.tiles, n,
                                                                        static_cast<T*>(dB), static_cast<T*>(dC));
  if ((rc = check_launch(who))) return rc;
  return column_sum(p.part_p, (long long)p.rows * p.nchunks, (long long)p.D * (p.N + 2), dparams, st, who);
}

}  // namespace scan
}  // namespace ttt

using namespace ttt;

static int bwd_pieces(int rows, int L, int D, int N) {
  scan::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.N = N;
  char dummy;
  scan::plan(p, &dummy, ~(size_t)0, 0, "");
  return p.nchunks;
}

extern "C" size_t ttt_selective_scan_bwd_scratch_bytes(int rows, int L, int D, int G, int N) {
  if (rows < 1 || L < 1 || D < 1 || G < 1 || N < 1 || N > scan::kMaxStates || D % G) return 0;
  const scan::BwdScratch s = scan::bwd_scratch(rows, L, D, G, N, bwd_pieces(rows, L, D, N));
  return 2 * s.part_bc + s.part_p + scan::plan_bytes(rows, L, D, N);
}

extern "C" int ttt_selective_scan_bwd(int rows, int L, int D, int G, int N, const void* u, const void* delta,
                                      const void* B, const void* C, const void* z, int dt, const long long* strides,
                                      const float* A, const float* Dskip, const float* delta_bias, int softplus,
                                      const int* seq, const float* init, const float* saved, const void* dout,
                                      const float* dfin, void* du, void* ddelta, void* dB, void* dC, void* dz,
                                      float* dinit, float* dparams, void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "ttt_selective_scan_bwd";
  int rc = scan::check_sizes(who, rows, L, D, G, N, dt);
  if (rc) return rc;
  TTT_REQUIRE(u && delta && B && C && A && strides && saved && dout && du && ddelta && dB && dC && dparams,
              TTT_ERR_NULL, "%s: NULL pointer argument", who);
  TTT_REQUIRE(!z == !dz, TTT_ERR_NULL, "%s: z and dz are given together", who);
  TTT_REQUIRE(!seq || rows == 1, TTT_ERR_SHAPE, "%s: packed sequences lie in one row, got %d", who, rows);
  scan::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.G = G, p.N = N, p.Dg = D / G;
  p.u = u, p.delta = delta, p.B = B, p.C = C, p.z = z;
  p.u_b = strides[0], p.u_l = strides[1], p.delta_b = strides[2], p.delta_l = strides[3];
  p.B_b = strides[4], p.B_l = strides[5], p.B_g = strides[6], p.C_b = strides[7], p.C_l = strides[8];
  p.C_g = strides[9], p.z_b = strides[10], p.z_l = strides[11];
  p.A = A, p.Dskip = Dskip, p.bias = delta_bias, p.softplus = softplus;
  p.seq = seq, p.init = init, p.hsave = const_cast<float*>(saved), p.dout = dout, p.dfin = dfin;
  p.du = du, p.ddelta = ddelta, p.dz = dz, p.dinit = dinit;
  const int every = scan::save_every(N);
  p.nsave = (L + every - 1) / every;
  p.quads = scan::quads(p, dt);
  const int nchunks = bwd_pieces(rows, L, D, N);
  const scan::BwdScratch s = scan::bwd_scratch(rows, L, D, G, N, nchunks);
  if ((rc = scan::plan(p, scratch, scratch_bytes, 2 * s.part_bc + s.part_p, who))) return rc;
  p.tiles = (int)s.tiles;
  p.part_B = static_cast<float*>(scratch);
  p.part_C = p.part_B + s.part_bc / sizeof(float);
  p.part_p = p.part_C + s.part_bc / sizeof(float);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.nchunks > 1 && (rc = scan::chunk_states(p, dt, true, st, who))) return rc;
  return dt == DT_BF16  ? scan::launch_bwd<__nv_bfloat16>(p, dB, dC, dparams, st, who)
         : dt == DT_F16 ? scan::launch_bwd<__half>(p, dB, dC, dparams, st, who)
                        : scan::launch_bwd<float>(p, dB, dC, dparams, st, who);
}
