// Selective state space scan, backward (the recurrence is in selective_scan.cuh):
//
//   dy = dout silu(z),  g[t] = C dy + a[t+1] g[t+1],  q = g a h[t-1]
//   dC = sum_d h dy,  dB = sum_d g dt u,  s1 = <g, B>,  s2 = <q, A>
//   du = dt s1 + D dy,  ddt = u s1 + s2,  dA = sum q dt,  dz = dout y silu'(z)
//
// A CTA walks its channels' time axis backwards in tiles of TB tokens. The forward kept the
// state before every SUB-th token; from there the states are run forward again with the decays
// a and a h[t-1] held in registers, then g runs back through them. Sums over a channel's
// states (s1, s2 and y) go through shared memory. Sums over channels (dB, dC) are products of
// the state matrix h (or g) of a token with its vector dy (or dt u), so the tensor cores take
// them: one mma.sync of 16 (states of two channel groups) x 4 (channels) per pair of states, the
// vector in the column of its token and zeros in the others. The factors have 11 bits there:
// for bf16 inputs they are rounded to that (2^-11 each, against 2^-8 of dB's and dC's own type),
// for fp16 and fp32 split in two such parts, three products a pair, 2^-21.
// What the CTAs of a group have of dB and dC, and what the rows and pieces have of dA, dD and
// dbias, is written as partials and added in a fixed order afterwards, so that results do not
// depend on timing.
#include "selective_scan.cuh"

namespace ttt {
namespace scan {

template <int LN, int NPT>
struct Bwd {
  static constexpr int THREADS = 256, WARPS = THREADS / 32;
  static constexpr int DT = THREADS / LN;     // channels of a CTA
  static constexpr int NP = LN * NPT;         // states, padded
  static constexpr int SUB = save_every_of(NPT);  // tokens whose states are in registers: save_every()
  static constexpr int TB = 2 * SUB;          // tokens of a tile
  static constexpr int CG = 8 / LN;           // groups of 4 channels in a warp
  static constexpr int TS = LN < SUB ? LN : SUB;  // tokens side by side in a product's columns
  static constexpr int TWOS = TB * DT / 2 / THREADS > 0 ? TB * DT / 2 / THREADS : 1;  // couples of a thread
  static constexpr int STEP = 2 * LN;         // tokens between them
  struct Smem {
    float B[TB * NP], C[TB * NP];
    float4 d[TB * DT];                        // step size twice, step size * input twice
    float2 dy[TB * DT];                       // twice
    float2 s12[TB * THREADS];
    float s3[TB * THREADS];
    float dB[WARPS * CG][TB * NP], dC[WARPS * CG][TB * NP];
    float2 red[THREADS];
    SeqMask m;
  };
};

__device__ __forceinline__ float tf32(float x) {
  unsigned r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}
__device__ __forceinline__ void mma_16x8x4(float (&c)[4], float a0, float a1, float b) {
  asm volatile("mma.sync.aligned.m16n8k4.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(b)));
}
// The 11 leading bits of x, for the split form: x = high + high(x - high) to 2^-21.
__device__ __forceinline__ float high(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// c += v b over the warp's channels, v a pair of states; SPLIT: both factors in two parts.
template <bool SPLIT>
__device__ __forceinline__ void add_product(float (&c)[4], float2 v, float b, float b_low) {
  if constexpr (SPLIT) {
    const float x = high(v.x), y = high(v.y);
    const float2 low = __fadd2_rn(v, make_float2(-x, -y));
    mma_16x8x4(c, high(low.x), high(low.y), b);
    mma_16x8x4(c, x, y, b_low);
    mma_16x8x4(c, x, y, b);
  } else {
    mma_16x8x4(c, tf32(v.x), tf32(v.y), b);
  }
}

template <typename T, int LN, int NPT, bool SEQ>
__global__ void __launch_bounds__(256, NPT == 4 ? 2 : 1) scan_bwd_kernel(const __grid_constant__ Params p) {
  using F = Bwd<LN, NPT>;
  constexpr bool SPLIT = !std::is_same<T, __nv_bfloat16>::value;
  constexpr int H = NPT / 2;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // lane -> channel and states, as the products' first operand wants them: rows lane / 4 are
  // (channel group, state run), columns lane % 4 the group's channels
  const int l3 = lane & 3, row8 = lane >> 2, cg = row8 / LN, nl = row8 % LN;
  const int cl = warp * (32 / LN) + l3 + 4 * cg, n0 = nl * NPT, at = cl * LN + nl;
  // and as the second operand wants them: column lane / 4 is (token, channel group)
  const int col_tok = row8 / F::CG, col_ch = warp * (32 / LN) + l3 + 4 * (row8 % F::CG);
  const int d = w.g * p.Dg + w.d0 + cl;
  const bool on = w.d0 + cl < p.Dg;
  // channels pd, pd + 1 and tokens tq, tq + STEP, .. of a tile in the element-wise passes
  const int pc = tid % (F::DT / 2) * 2, tq = tid / (F::DT / 2), pd = w.g * p.Dg + w.d0 + pc;
  const bool on0 = w.d0 + pc < p.Dg, on1 = w.d0 + pc + 1 < p.Dg;
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const long long DN = (long long)p.D * p.N;
  const int* seq = SEQ ? p.seq : nullptr;

  float hs[NPT];
  load_states<NPT>(p.A, d, n0, p.N, on, hs);
#pragma unroll
  for (int i = 0; i < NPT; ++i) hs[i] *= kLog2e;
  const Pairs<NPT> A2 = pairs_of<NPT>(hs);
  if (p.nchunks > 1)
    load_states<NPT>(p.cstate + ((long long)w.row * p.nchunks + w.piece) * DN, d, n0, p.N, on, hs);
  else
    load_states<NPT>(p.dfin + w.row * DN, d, n0, p.N, on && p.dfin && !SEQ, hs);
  Pairs<NPT> carry = pairs_of<NPT>(hs), dA;
#pragma unroll
  for (int j = 0; j < H; ++j) dA.v[j] = make_float2(0.f, 0.f);
  const float2 skip = params_of(p.Dskip, pd, on0, on1), bias = params_of(p.bias, pd, on0, on1);
  const T* u = static_cast<const T*>(p.u) + w.row * p.u_b + pd;
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + pd;
  const T* z = static_cast<const T*>(p.z) + w.row * p.z_b + pd;
  const T* dout = static_cast<const T*>(p.dout) + (long long)w.row * p.L * p.D + pd;
  const T* B = static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const T* C = static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g;
  const long long row0 = (long long)w.row * p.L;
  const float* kept = p.hsave + (long long)w.row * p.nsave * DN;
  float2 sum_D = all2(0.f), sum_bias = all2(0.f);

  for (int tile = (tend - 1) / F::TB; tile >= tbeg / F::TB; --tile) {
    const int t0 = tile * F::TB;
    Two<T> uu[F::TWOS], rr[F::TWOS], zz[F::TWOS], dd[F::TWOS];
    if (SEQ) stage_masks<F::TB>(&s.m, p.seq, t0, tend, p.L);
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = tq + k * F::STEP, tok = t0 + t;
      const bool in = t < F::TB && tok < tend && in_sequence(seq, tok), i0 = in && on0, i1 = in && on1;
      uu[k] = load_two(u + tok * p.u_l, i0, i1, p.couples), rr[k] = load_two(delta + tok * p.delta_l, i0, i1, p.couples);
      dd[k] = load_two(dout + (long long)tok * p.D, i0, i1, p.couples);
      zz[k] = load_two(z + tok * p.z_l, i0 && p.z, i1 && p.z, p.couples);
    }
    // the states before the tile's halves
    float h_kept[2][NPT];
#pragma unroll
    for (int half = 0; half < 2; ++half)
      load_states<NPT>(kept + (2 * tile + half) * DN, d, n0, p.N, on && t0 + half * F::SUB < tend, h_kept[half]);
    stage_rows<T, F::NP, F::TB, F::THREADS>(s.B, B, p.B_l, t0, tend, p.N, seq, p.quads);
    stage_rows<T, F::NP, F::TB, F::THREADS>(s.C, C, p.C_l, t0, tend, p.N, seq, p.quads);
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = tq + k * F::STEP, tok = t0 + t;
      if (t < F::TB) {
        float2 dt = __fadd2_rn(two_f(rr[k]), bias), dy = two_f(dd[k]);
        if (p.softplus) dt = softplus2(dt);
        if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
        const float2 x = __fmul2_rn(dt, two_f(uu[k]));
        if (p.z) dy = __fmul2_rn(dy, silu2(two_f(zz[k])));
        s.d[t * F::DT + pc] = make_float4(dt.x, dt.x, x.x, x.x), s.d[t * F::DT + pc + 1] = make_float4(dt.y, dt.y, x.y, x.y);
        *reinterpret_cast<float4*>(&s.dy[t * F::DT + pc]) = make_float4(dy.x, dy.x, dy.y, dy.y);
      }
    }
    __syncthreads();

#pragma unroll 1
    for (int half = 1; half >= 0; --half) {
      const int b = half * F::SUB;
      if (t0 + b >= tend) continue;
      const auto tokens = [&](auto checks) {
        float2 a[F::SUB][H], ah[F::SUB][H];
        Pairs<NPT> h;
#pragma unroll
        for (int i = 0; i < NPT; ++i) hs[i] = half ? h_kept[1][i] : h_kept[0][i];
        h = pairs_of<NPT>(hs);
#pragma unroll
        for (int k = 0; k < F::SUB; ++k) {
          const int t = b + k;
          if constexpr (decltype(checks)::value) {
            if (SEQ && (s.m.start >> t & 1)) {
              const int sq = p.seq[t0 + t];
              load_states<NPT>(p.init + sq * DN, d, n0, p.N, on && sq >= 0 && p.init, hs);
              h = pairs_of<NPT>(hs);
            }
          }
          const float4 dd4 = s.d[t * F::DT + cl];
          const float2 dt = make_float2(dd4.x, dd4.y), dtu = make_float2(dd4.z, dd4.w);
          const Pairs<NPT> B2 = row_pairs<NPT>(s.B + t * F::NP + n0);
#pragma unroll
          for (int j = 0; j < H; ++j) {
            a[k][j] = decay(dt, A2.v[j]);
            ah[k][j] = __fmul2_rn(a[k][j], h.v[j]);
            h.v[j] = __ffma2_rn(dtu, B2.v[j], ah[k][j]);
          }
        }
        // tokens of two sequences never share a product: a NaN of one would reach the other's columns
        constexpr int TS = decltype(checks)::value ? 1 : F::TS;
        Pairs<NPT> dA_here;
#pragma unroll
        for (int j = 0; j < H; ++j) dA_here.v[j] = make_float2(0.f, 0.f);
#pragma unroll
        for (int g0 = F::SUB - TS; g0 >= 0; g0 -= TS) {
          float accB[H][4], accC[H][4];
#pragma unroll
          for (int j = 0; j < H; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) accB[j][e] = accC[j][e] = 0.f;
          float vB = 0.f, vC = 0.f;  // the products' vectors, in this lane's token and channel
          if (col_tok < TS) {
            vB = s.d[(b + g0 + col_tok) * F::DT + col_ch].z;
            vC = s.dy[(b + g0 + col_tok) * F::DT + col_ch].x;
          }
          const float hB = SPLIT ? high(vB) : tf32(vB), hC = SPLIT ? high(vC) : tf32(vC);
          const float lB = SPLIT ? high(vB - hB) : 0.f, lC = SPLIT ? high(vC - hC) : 0.f;
#pragma unroll
          for (int k = g0 + TS - 1; k >= g0; --k) {
            const int t = b + k;
            if constexpr (decltype(checks)::value) {
              if (t0 + t >= tend) continue;
              if (SEQ && (s.m.end >> t & 1)) {
                const int sq = p.seq[t0 + t];
                load_states<NPT>(p.dfin + sq * DN, d, n0, p.N, on && sq >= 0 && p.dfin, hs);
                carry = pairs_of<NPT>(hs);
              }
            }
            const float4 dd4 = s.d[t * F::DT + cl];
            const float2 dt = make_float2(dd4.x, dd4.y), dtu = make_float2(dd4.z, dd4.w), dy = s.dy[t * F::DT + cl];
            const Pairs<NPT> B2 = row_pairs<NPT>(s.B + t * F::NP + n0), C2 = row_pairs<NPT>(s.C + t * F::NP + n0);
            const bool mine = col_tok == k - g0;
            const float bB = mine ? hB : 0.f, bC = mine ? hC : 0.f;
            const float cB = SPLIT && mine ? lB : 0.f, cC = SPLIT && mine ? lC : 0.f;
            float2 s1 = make_float2(0.f, 0.f), s2 = s1, s3 = s1;
#pragma unroll
            for (int j = 0; j < H; ++j) {
              const float2 g = __ffma2_rn(C2.v[j], dy, carry.v[j]), hn = __ffma2_rn(dtu, B2.v[j], ah[k][j]);
              const float2 q = __fmul2_rn(g, ah[k][j]);
              s1 = __ffma2_rn(g, B2.v[j], s1), s2 = __ffma2_rn(q, A2.v[j], s2), s3 = __ffma2_rn(hn, C2.v[j], s3);
              dA_here.v[j] = __ffma2_rn(q, dt, dA_here.v[j]);
              carry.v[j] = __fmul2_rn(a[k][j], g);
              add_product<SPLIT>(accB[j], g, bB, cB);
              add_product<SPLIT>(accC[j], hn, bC, cC);
            }
            s.s12[t * F::THREADS + at] = make_float2(s1.x + s1.y, s2.x + s2.y);
            s.s3[t * F::THREADS + at] = s3.x + s3.y;
            if constexpr (decltype(checks)::value) {
              if (SEQ && p.dinit && (s.m.start >> t & 1)) {
                const int sq = p.seq[t0 + t];
                unpair(carry, hs);
                store_states<NPT>(p.dinit + sq * DN, d, n0, p.N, on && sq >= 0, hs);
              }
            }
          }
          // of the products' two columns in this lane, those of the row's own channel group
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = 2 * l3 + e, tc = c / F::CG;
            if (c % F::CG == cg && tc < TS) {
              const int o = (b + g0 + tc) * F::NP + n0;
#pragma unroll
              for (int j = 0; j < H; ++j) {
                *reinterpret_cast<float2*>(&s.dB[warp * F::CG + cg][o + 2 * j]) = make_float2(accB[j][e], accB[j][2 + e]);
                *reinterpret_cast<float2*>(&s.dC[warp * F::CG + cg][o + 2 * j]) = make_float2(accC[j][e], accC[j][2 + e]);
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < H; ++j) dA.v[j] = __fadd2_rn(dA.v[j], dA_here.v[j]);
      };
      if (t0 + b + F::SUB > tend || (SEQ && ((s.m.start | s.m.end) >> b & ((1u << F::SUB) - 1))))
        tokens(std::true_type{});
      else tokens(std::false_type{});
    }
    __syncthreads();

#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = tq + k * F::STEP, tok = t0 + t;
      if (t < F::TB && tok < tend && on0) {
        // sums over the states: s1, s2 of the two channels, then y
        float4 s12 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < LN; ++j) {
          const float2 x = s.s12[t * F::THREADS + pc * LN + j], y = s.s12[t * F::THREADS + (pc + 1) * LN + j];
          s12.x += x.x, s12.y += y.x, s12.z += x.y, s12.w += y.y;
        }
        const float2 s1 = make_float2(s12.x, s12.y), s2 = make_float2(s12.z, s12.w);
        const float2 s3 = state_sums<LN>(s.s3 + t * F::THREADS + pc * LN);
        const float2 dt = make_float2(s.d[t * F::DT + pc].x, s.d[t * F::DT + pc + 1].x), uv = two_f(uu[k]);
        const float2 dy = make_float2(s.dy[t * F::DT + pc].x, s.dy[t * F::DT + pc + 1].x);
        float2 du = __ffma2_rn(dt, s1, __fmul2_rn(skip, dy)), ddt = __ffma2_rn(uv, s1, __fmul2_rn(s2, all2(kLn2)));
        float2 dz = all2(0.f);
        if (p.softplus) ddt = __fmul2_rn(ddt, sigmoid2(__fadd2_rn(two_f(rr[k]), bias)));
        if (p.z) {  // silu'(g) = s (1 + g (1 - s))
          const float2 g = two_f(zz[k]), sg = sigmoid2(g);
          const float2 slope = __fmul2_rn(sg, __ffma2_rn(g, __fadd2_rn(all2(1.f), neg2(sg)), all2(1.f)));
          dz = __fmul2_rn(__fmul2_rn(two_f(dd[k]), slope), __ffma2_rn(skip, uv, s3));
        }
        if (SEQ && !(s.m.in >> t & 1)) du = ddt = dz = all2(0.f);  // a token of no sequence
        else sum_D = __ffma2_rn(uv, dy, sum_D), sum_bias = __fadd2_rn(sum_bias, ddt);
        const long long o = (row0 + tok) * p.D + pd;
        store_two(static_cast<T*>(p.du) + o, du, true, on1, p.couples);
        store_two(static_cast<T*>(p.ddelta) + o, ddt, true, on1, p.couples);
        if (p.z) store_two(static_cast<T*>(p.dz) + o, dz, true, on1, p.couples);
      }
    }
    const int tile_g = w.d0 / F::DT;
    for (int i = tid; i < F::TB * F::NP; i += F::THREADS) {
      const int t = i / F::NP, n = i - t * F::NP;
      if (t0 + t < tend && n < p.N) {
        float vb = 0.f, vc = 0.f;
#pragma unroll
        for (int k = 0; k < F::WARPS * F::CG; ++k) vb += s.dB[k][i], vc += s.dC[k][i];
        const bool out = SEQ && !(s.m.in >> t & 1);
        const long long o = (((long long)tile_g * p.rows * p.L + row0 + t0 + t) * p.G + w.g) * p.N + n;
        p.part_B[o] = out ? 0.f : vb, p.part_C[o] = out ? 0.f : vc;
      }
    }
    __syncthreads();
  }

  unpair(carry, hs);
  if (p.dinit && !SEQ && tbeg == 0) store_states<NPT>(p.dinit + w.row * DN, d, n0, p.N, on, hs);
  float* part = p.part_p + ((long long)w.row * p.nchunks + w.piece) * p.D * (p.N + 2);
  unpair(dA, hs);
  store_states<NPT>(part, d, n0, p.N, on, hs);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    s.red[tid] = k ? sum_bias : sum_D;
    __syncthreads();
    if (tid < F::DT / 2) {
      float2 v = all2(0.f);
#pragma unroll
      for (int j = 0; j < F::STEP; ++j) v = __fadd2_rn(v, s.red[tid + j * (F::DT / 2)]);
      if (on0) part[DN + (long long)k * p.D + pd] = v.x;
      if (on1) part[DN + (long long)k * p.D + pd + 1] = v.y;
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
    constexpr int LN = decltype(ln)::value, NPT = decltype(npt)::value;
    auto kernel = p.seq ? scan_bwd_kernel<T, LN, NPT, true> : scan_bwd_kernel<T, LN, NPT, false>;
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
  p.quads = scan::quads(p, dt), p.couples = scan::couples(p, dt);
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
