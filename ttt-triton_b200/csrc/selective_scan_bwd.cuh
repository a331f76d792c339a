// Selective state space scan, backward: the kernels (the recurrence is in selective_scan.cuh).
//
//   dy = dout silu(z),  g[t] = C dy + a[t+1] g[t+1],  q = g a h[t-1]
//   dC = sum_d h dy,  dB = sum_d g dt u,  s1 = <g, B>,  s2 = <q, A>
//   du = dt s1 + D dy,  ddt = u s1 + s2,  dA = sum q dt,  dz = dout y silu'(z)
//
// A CTA walks its channels' time axis backwards in tiles of SUB tokens. The forward kept the
// state before each; from there the first part of the CTA runs the tile's states forward again
// with the decays a and a h[t-1] held in registers, then g back through them, two channels a
// thread. Meanwhile the second part finishes the element-wise gradients of the tile before and
// prepares the step sizes and gates of the next (one barrier a tile). Sums over a channel's
// states (s1, s2 and y) pass through shared memory. Sums over channels (dB, dC): a thread adds
// its two channels' products, the four threads that have the same states exchange theirs, and
// the second part adds what warps and groups of lanes have. All in fp32, so that no token's
// value meets another's: on the tensor cores, with one token a column, a non-finite value spoils
// the columns beside it (zero times infinity), 16-bit operands need two or three parts, and the
// conversions cost more than the exchanges: 16 x 2048 x 1536, 16 states, 1.19 ms against 1.27
// (bf16 parts to 2^-17) and 1.55 (exact); 64 states 4 x 2048 x 1024 725 us against 827.
// What the CTAs of a group have of dB and dC, and
// what the rows and pieces have of dA, dD and dbias, is written as partials and added in a
// fixed order afterwards, so that results do not depend on timing.
#pragma once

#include "selective_scan.cuh"

namespace ttt {
namespace scan {

template <int LN, int NPT>
struct Bwd {
  static constexpr int MAIN = 128, HELP = 128, THREADS = MAIN + HELP;  // threads of the two parts
  static constexpr int WARPS = MAIN / 32;
  static constexpr int CW = 64 / LN, DT = WARPS * CW;  // channels of a warp and of a CTA
  static constexpr int NP = LN * NPT;                // states, padded
  static constexpr int SUB = save_every_of(NPT);     // tokens whose states are in registers
  static constexpr int RING = 4;                     // runs whose first states are on their way
  static constexpr int RUNS = LN >= 4 ? 2 : 1, TB = RUNS * SUB;  // tokens of a tile
  static constexpr int CG = 8 / LN;                  // groups of 8 channels in a warp
  static constexpr int STEP = HELP / (DT / 2);       // tokens between a thread's couples of channels
  static constexpr int TWOS = (TB + STEP - 1) / STEP;
  static constexpr int YS = DT + (LN == 1 ? 0 : LN == 2 ? 16 : 8);  // row of partial sums, padded off bank conflicts
  struct Tile {
    float B[TB * NP], C[TB * NP];
    float2 d[TB * DT];                               // step size, step size * input
    float dy[TB * DT];
    float s1[TB * LN * YS], s2[TB * LN * YS], s3[TB * LN * YS];
    float sums[2 * WARPS * CG * TB * NP];            // over a group's channels: dB of all groups, dC of all
  };
  struct Smem {
    Tile tile[2];
    float2 dA[MAIN * NPT], dD[HELP], dbias[HELP];    // sums over many tiles
    float4 kept[RING][MAIN * NPT / 2];               // states before the coming runs, each thread's own
  };
};

// Adds a token's products for dB and dC over the 4 threads of a channel group (the lanes that differ
// in their last two bits), two exchanges that halve what a thread holds: it ends with the H / 2 pairs
// of states from (l3 & 1) H / 2 on, of dB (l3 < 2) or dC.
template <int H>
__device__ __forceinline__ void add_over_channels(const float2 (&vB)[H], const float2 (&vC)[H], int l3, float2 (&sum)[H / 2]) {
  const auto other = [](float2 x, int lanes) {
    return make_float2(__shfl_xor_sync(0xffffffffu, x.x, lanes), __shfl_xor_sync(0xffffffffu, x.y, lanes));
  };
  float2 half[H];
#pragma unroll
  for (int j = 0; j < H; ++j) half[j] = __fadd2_rn(l3 & 2 ? vC[j] : vB[j], other(l3 & 2 ? vB[j] : vC[j], 2));
#pragma unroll
  for (int j = 0; j < H / 2; ++j)
    sum[j] = __fadd2_rn(l3 & 1 ? half[j + H / 2] : half[j], other(l3 & 1 ? half[j] : half[j + H / 2], 1));
}

// Barrier ID of the CTA's first THREADS (or of its second part), waited for at places of its own.
template <int ID, int THREADS>
__device__ __forceinline__ void part_barrier() {
  asm volatile("barrier.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory");
}

template <typename T, int LN, int NPT, bool SEQ, bool TWO>
__global__ void __launch_bounds__(256, NPT == 4 ? 2 : 1) scan_bwd_kernel(const __grid_constant__ Params p) {
  using F = Bwd<LN, NPT>;
  constexpr int H = NPT / 2;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  auto& s = *reinterpret_cast<typename F::Smem*>(raw_smem);
  const Where w = where<F::DT>(p);
  const int tbeg = w.piece * p.chunk, tend = min(p.L, tbeg + p.chunk);
  const int last = (tend - 1) / F::TB, ntiles = last - tbeg / F::TB + 1;  // tile i is tokens (last - i) TB ..
  const long long DN = (long long)p.D * p.N;
  float* const part = p.part_p + ((long long)w.row * p.nchunks + w.piece) * p.D * (p.N + 2);

  if (threadIdx.x < F::MAIN) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // lane -> states and channels, as the sums over channels want them: lane / 4 is (channel
    // group, run of states), lane % 4 one of the threads whose sums are added
    const int l3 = lane & 3, row8 = lane >> 2, cg = row8 / LN, nl = row8 % LN, n0 = nl * NPT;
    const int cl = warp * F::CW + 8 * cg + 2 * l3;
    // where this thread's part of a token's sums over channels lies
    const int sums = ((l3 >> 1) * F::WARPS * F::CG + warp * F::CG + cg) * F::TB * F::NP + n0 + (l3 & 1) * H;
    const int d = w.g * p.Dg + w.d0 + cl;
    const bool c0 = w.d0 + cl < p.Dg, c1 = w.d0 + cl + 1 < p.Dg;
    const float* kept = p.hsave + (long long)w.row * p.nsave * DN;
    const auto load2 = [&](const float* base, bool on) { return load_both<NPT>(base, d, n0, p.N, on && c0, on && c1); };

    Both<NPT> A2 = load2(p.A, true);
    Both<NPT> carry = p.nchunks > 1 ? load2(p.cstate + ((long long)w.row * p.nchunks + w.piece) * DN, true)
                                    : load2(p.dfin + w.row * DN, p.dfin && !SEQ);
    // The states that the forward kept come by asynchronous copies, RING - 1 runs ahead: fetched
    // into registers they would have to be waited for early. Each thread copies its own.
    const bool whole = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.hsave) & 15) == 0;
    const auto fetch_states = [&](int run) {
      if (run * F::SUB >= tbeg) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float* src = kept + run * DN + (long long)(d + c) * p.N + n0;
          const bool on = c ? c1 : c0;
#pragma unroll
          for (int e = 0; e < NPT / 4; ++e) {
            float4* dst = &s.kept[run % F::RING][tid + (c * (NPT / 4) + e) * F::MAIN];
            const int n = n0 + 4 * e;
            if (whole) {
              const bool in = on && n < p.N;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(dst)),
                           "l"(in ? src + 4 * e : kept), "r"(in ? 16 : 0));
            } else {
              float x[4];
#pragma unroll
              for (int f = 0; f < 4; ++f) x[f] = on && n + f < p.N ? src[4 * e + f] : 0.f;
              *dst = make_float4(x[0], x[1], x[2], x[3]);
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;");
    };
    int run = (tend - 1) / F::SUB;  // the run that comes next
#pragma unroll
    for (int k = 0; k < F::RING - 1; ++k) fetch_states(run - k);
    Both<NPT> dA;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        A2.c[c].v[j] = __fmul2_rn(A2.c[c].v[j], all2(kLog2e)), dA.c[c].v[j] = all2(0.f);
        s.dA[tid + (c * H + j) * F::MAIN] = all2(0.f);
      }

    for (int i = 0; i < ntiles; ++i) {
      part_barrier<1, F::THREADS>();
      auto& tile = s.tile[i & 1];
      const int tt = (last - i) * F::TB;
      SeqMask mask{};
      if (SEQ) mask = warp_masks<F::TB>(p.seq, tt, tend, p.L);
#pragma unroll 1
      for (int t0 = tt + (F::RUNS - 1) * F::SUB; t0 >= tt; t0 -= F::SUB) {
        if (t0 >= tend) continue;
        const int b = t0 - tt;
        const auto tokens = [&](auto checks) {
          constexpr bool CHECK = decltype(checks)::value;
          float2 a[F::SUB][2][H], ah[F::SUB][2][H];
          asm volatile("cp.async.wait_group %0;" ::"n"(F::RING - 2) : "memory");
          Both<NPT> h;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < NPT / 4; ++e) {
              const float4 q = s.kept[run % F::RING][tid + (c * (NPT / 4) + e) * F::MAIN];
              h.c[c].v[2 * e] = make_float2(q.x, q.y), h.c[c].v[2 * e + 1] = make_float2(q.z, q.w);
            }
          fetch_states(run - (F::RING - 1));
          --run;
#pragma unroll
          for (int k = 0; k < F::SUB; ++k) {
            if constexpr (CHECK && SEQ) {
              if (mask.start >> (b + k) & 1) {
                const int sq = p.seq[t0 + k];
                h = load2(p.init + sq * DN, sq >= 0 && p.init);
              }
            }
            const float4 d4 = *reinterpret_cast<const float4*>(&tile.d[(b + k) * F::DT + cl]);
            const Pairs<NPT> B2 = row_pairs<NPT>(tile.B + (b + k) * F::NP + n0);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < H; ++j) {
                a[k][c][j] = decay(all2(c ? d4.z : d4.x), A2.c[c].v[j]);
                ah[k][c][j] = __fmul2_rn(a[k][c][j], h.c[c].v[j]);
                h.c[c].v[j] = __ffma2_rn(all2(c ? d4.w : d4.y), B2.v[j], ah[k][c][j]);
              }
          }
#pragma unroll
          for (int k = F::SUB - 1; k >= 0; --k) {
            if constexpr (CHECK) {
              if (t0 + k >= tend) continue;
              if (SEQ && (mask.end >> (b + k) & 1)) {
                const int sq = p.seq[t0 + k];
                carry = load2(p.dfin + sq * DN, sq >= 0 && p.dfin);
              }
            }
            const float4 d4 = *reinterpret_cast<const float4*>(&tile.d[(b + k) * F::DT + cl]);
            const float2 dy2 = *reinterpret_cast<const float2*>(&tile.dy[(b + k) * F::DT + cl]);
            const Pairs<NPT> B2 = row_pairs<NPT>(tile.B + (b + k) * F::NP + n0), C2 = row_pairs<NPT>(tile.C + (b + k) * F::NP + n0);
            const float2 zero = all2(0.f);
            float2 vB[H], vC[H], s1[2] = {zero, zero}, s2[2] = {zero, zero}, s3[2] = {zero, zero};
#pragma unroll
            for (int j = 0; j < H; ++j) {
              float2 g[2], hn[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const float2 ahj = ah[k][c][j];
                g[c] = __ffma2_rn(C2.v[j], all2(c ? dy2.y : dy2.x), carry.c[c].v[j]);
                hn[c] = __ffma2_rn(all2(c ? d4.w : d4.y), B2.v[j], ahj);
                const float2 q = __fmul2_rn(g[c], ahj);
                s1[c] = j ? __ffma2_rn(g[c], B2.v[j], s1[c]) : __fmul2_rn(g[c], B2.v[j]);
                s2[c] = j ? __ffma2_rn(q, A2.c[c].v[j], s2[c]) : __fmul2_rn(q, A2.c[c].v[j]);
                s3[c] = j ? __ffma2_rn(hn[c], C2.v[j], s3[c]) : __fmul2_rn(hn[c], C2.v[j]);
                dA.c[c].v[j] = __ffma2_rn(q, all2(c ? d4.z : d4.x), dA.c[c].v[j]);
                carry.c[c].v[j] = __fmul2_rn(a[k][c][j], g[c]);
              }
              vB[j] = __ffma2_rn(g[0], all2(d4.y), __fmul2_rn(g[1], all2(d4.w)));
              vC[j] = __ffma2_rn(hn[0], all2(dy2.x), __fmul2_rn(hn[1], all2(dy2.y)));
            }
            float2 sum[H / 2];
            add_over_channels<H>(vB, vC, l3, sum);
#pragma unroll
            for (int j = 0; j < H / 2; ++j)
              *reinterpret_cast<float2*>(&tile.sums[sums + (b + k) * F::NP + 2 * j]) = sum[j];
            const int o = ((b + k) * LN + nl) * F::YS + cl;
            *reinterpret_cast<float2*>(&tile.s1[o]) = make_float2(s1[0].x + s1[0].y, s1[1].x + s1[1].y);
            *reinterpret_cast<float2*>(&tile.s2[o]) = make_float2(s2[0].x + s2[0].y, s2[1].x + s2[1].y);
            *reinterpret_cast<float2*>(&tile.s3[o]) = make_float2(s3[0].x + s3[0].y, s3[1].x + s3[1].y);
            if constexpr (CHECK && SEQ) {
              if (p.dinit && (mask.start >> (b + k) & 1)) {
                const int sq = p.seq[t0 + k];
                store_both<NPT>(p.dinit + sq * DN, d, n0, p.N, sq >= 0 && c0, sq >= 0 && c1, carry);
              }
            }
          }
        };
        if (t0 + F::SUB > tend || (SEQ && ((mask.start | mask.end) >> b & ((1u << F::SUB) - 1)))) tokens(std::true_type{});
        else tokens(std::false_type{});
      }
      if (i % 8 == 7 || i + 1 == ntiles) {  // short sums first: a long chain of additions loses bits
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < H; ++j) {
            float2& total = s.dA[tid + (c * H + j) * F::MAIN];
            total = __fadd2_rn(total, dA.c[c].v[j]);
            dA.c[c].v[j] = all2(0.f);
          }
      }
    }
    part_barrier<1, F::THREADS>();
    if (p.dinit && !SEQ && tbeg == 0) store_both<NPT>(p.dinit + w.row * DN, d, n0, p.N, c0, c1, carry);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < H; ++j) dA.c[c].v[j] = s.dA[tid + (c * H + j) * F::MAIN];
    store_both<NPT>(part, d, n0, p.N, c0, c1, dA);
    return;
  }

  const int tid = threadIdx.x - F::MAIN;
  const int* seq = SEQ ? p.seq : nullptr;
  // channels pd, pd + 1 at tokens tq, tq + STEP, .. of a tile
  const int pc = tid % (F::DT / 2) * 2, tq = tid / (F::DT / 2), pd = w.g * p.Dg + w.d0 + pc;
  const bool on0 = w.d0 + pc < p.Dg, on1 = w.d0 + pc + 1 < p.Dg;
  const float2 skip = params_of(p.Dskip, pd, on0, on1), bias = params_of(p.bias, pd, on0, on1);
  float2 sum_D = all2(0.f), sum_bias = sum_D;
  s.dD[tid] = s.dbias[tid] = sum_D;
  const long long row0 = (long long)w.row * p.L, t_last = (long long)last * F::TB + tq;
  const T* u = static_cast<const T*>(p.u) + w.row * p.u_b + t_last * p.u_l + pd;
  const T* delta = static_cast<const T*>(p.delta) + w.row * p.delta_b + t_last * p.delta_l + pd;
  const T* z = static_cast<const T*>(p.z) + w.row * p.z_b + t_last * p.z_l + pd;
  const T* dout = static_cast<const T*>(p.dout) + (row0 + t_last) * p.D + pd;
  const long long o_last = (row0 + t_last) * p.D + pd, o_step = (long long)F::STEP * p.D;
  T* du = static_cast<T*>(p.du) + o_last;
  T* ddelta = static_cast<T*>(p.ddelta) + o_last;
  T* dz = static_cast<T*>(p.dz) + o_last;
  const long long u_step = F::STEP * p.u_l, delta_step = F::STEP * p.delta_l, z_step = F::STEP * p.z_l;
  const T* B = static_cast<const T*>(p.B) + w.row * p.B_b + w.g * p.B_g;
  const T* C = static_cast<const T*>(p.C) + w.row * p.C_b + w.g * p.C_g;
  float *part_B, *part_C;  // this thread's first value of the last tile
  {
    const long long o = (((long long)(w.d0 / F::DT) * p.rows * p.L + row0 + (long long)last * F::TB) * p.G + w.g) * p.N;
    part_B = p.part_B + o, part_C = p.part_C + o;
  }
  const long long part_step = (long long)p.G * p.N;  // from one token to the next
  // activations of a tile: fetched an interval before it is prepared, kept until its outputs
  struct Raw {
    Two<T> u, delta, z, dout;
  };
  Raw r2[F::TWOS], r1[F::TWOS], r0[F::TWOS];  // of tiles i + 2, i + 1 and i - 1 (i, once that is finished)
  Rows<T, F::NP, F::TB, F::HELP> rB, rC;
  const auto fetch = [&](int i) {  // tile i; called for 0, 1, ..
    const int tn = (last - i) * F::TB;
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) {
      const int t = tq + k * F::STEP;
      const bool in = t < F::TB && tn + t < tend && in_sequence(seq, tn + t), i0 = in && on0, i1 = in && on1;
      r2[k].u = load_two(u + k * u_step, i0, i1, TWO), r2[k].delta = load_two(delta + k * delta_step, i0, i1, TWO);
      r2[k].dout = load_two(dout + k * o_step, i0, i1, TWO);
      r2[k].z = load_two(z + k * z_step, i0 && p.z, i1 && p.z, TWO);
    }
    u -= F::TB * p.u_l, delta -= F::TB * p.delta_l, z -= F::TB * p.z_l, dout -= (long long)F::TB * p.D;
    rB.fetch(tid, B, p.B_l, tn, tend, seq, p.quads), rC.fetch(tid, C, p.C_l, tn, tend, seq, p.quads);
  };
  fetch(0);
  for (int i = -1; i <= ntiles; ++i) {
    const int tn = (last - i - 1) * F::TB, tl = (last - i + 1) * F::TB;
    auto& tile = s.tile[(i + 1) & 1];  // of tile i - 1, then of tile i + 1
    if (i >= 1) {
#pragma unroll
      for (int k = 0; k < F::TWOS; ++k) {
        const int t = tq + k * F::STEP, tok = tl + t;
        if (t < F::TB && tok < tend && on0) {
          float2 s1 = all2(0.f), s2 = s1, s3 = s1;
#pragma unroll
          for (int j = 0; j < LN; ++j) {
            const int o = (t * LN + j) * F::YS + pc;
            s1 = __fadd2_rn(s1, *reinterpret_cast<const float2*>(&tile.s1[o]));
            s2 = __fadd2_rn(s2, *reinterpret_cast<const float2*>(&tile.s2[o]));
            s3 = __fadd2_rn(s3, *reinterpret_cast<const float2*>(&tile.s3[o]));
          }
          const float4 d4 = *reinterpret_cast<const float4*>(&tile.d[t * F::DT + pc]);
          const float2 dt = make_float2(d4.x, d4.z), uv = two_f(r0[k].u);
          const float2 dy = *reinterpret_cast<const float2*>(&tile.dy[t * F::DT + pc]);
          float2 gu = __ffma2_rn(dt, s1, __fmul2_rn(skip, dy)), gd = __ffma2_rn(uv, s1, __fmul2_rn(s2, all2(kLn2)));
          float2 gz = all2(0.f);
          if (p.softplus) gd = __fmul2_rn(gd, sigmoid2(__fadd2_rn(two_f(r0[k].delta), bias)));
          if (p.z) {  // silu'(g) = s (1 + g (1 - s))
            const float2 g = two_f(r0[k].z), sg = sigmoid2(g);
            const float2 slope = __fmul2_rn(sg, __ffma2_rn(g, __fadd2_rn(all2(1.f), neg2(sg)), all2(1.f)));
            gz = __fmul2_rn(__fmul2_rn(two_f(r0[k].dout), slope), __ffma2_rn(skip, uv, s3));
          }
          if (SEQ && seq[tok] < 0) gu = gd = gz = all2(0.f);  // a token of no sequence
          else sum_D = __ffma2_rn(uv, dy, sum_D), sum_bias = __fadd2_rn(sum_bias, gd);
          store_two(du + k * o_step, gu, true, on1, TWO);
          store_two(ddelta + k * o_step, gd, true, on1, TWO);
          if (p.z) store_two(dz + k * o_step, gz, true, on1, TWO);
        }
      }
      du -= (long long)F::TB * p.D, ddelta -= (long long)F::TB * p.D, dz -= (long long)F::TB * p.D;
#pragma unroll
      for (int k = tid; k < F::TB * F::NP; k += F::HELP) {
        const int t = k / F::NP, n = k - t * F::NP;
        if (tl + t < tend && n < p.N) {
          float vb = 0.f, vc = 0.f;
#pragma unroll
          for (int e = 0; e < F::WARPS * F::CG; ++e)
            vb += tile.sums[e * F::TB * F::NP + k], vc += tile.sums[(F::WARPS * F::CG + e) * F::TB * F::NP + k];
          if (SEQ && seq[tl + t] < 0) vb = vc = 0.f;
          part_B[t * part_step + n] = vb, part_C[t * part_step + n] = vc;
        }
      }
      part_B -= F::TB * part_step, part_C -= F::TB * part_step;
      if (i % 8 == 0 || i == ntiles) {  // short sums first, as for dA
        s.dD[tid] = __fadd2_rn(s.dD[tid], sum_D), s.dbias[tid] = __fadd2_rn(s.dbias[tid], sum_bias);
        sum_D = sum_bias = all2(0.f);
      }
    }
#pragma unroll
    for (int k = 0; k < F::TWOS; ++k) r0[k] = r1[k], r1[k] = r2[k];
    if (i + 1 < ntiles) {
#pragma unroll
      for (int k = 0; k < F::TWOS; ++k) {
        const int t = tq + k * F::STEP, tok = tn + t;
        if (t < F::TB) {
          float2 dt = __fadd2_rn(two_f(r1[k].delta), bias), dy = two_f(r1[k].dout);
          if (p.softplus) dt = softplus2(dt);
          if (!(tok < tend && in_sequence(seq, tok))) dt = all2(0.f);
          const float2 x = __fmul2_rn(dt, two_f(r1[k].u));
          if (p.z) dy = __fmul2_rn(dy, silu2(two_f(r1[k].z)));
          *reinterpret_cast<float4*>(&tile.d[t * F::DT + pc]) = make_float4(dt.x, x.x, dt.y, x.y);
          *reinterpret_cast<float2*>(&tile.dy[t * F::DT + pc]) = dy;
        }
      }
      rB.put(tid, tile.B, B, p.B_l, tn, tend, p.N, seq, p.quads), rC.put(tid, tile.C, C, p.C_l, tn, tend, p.N, seq, p.quads);
      if (i + 2 < ntiles) fetch(i + 2);
    }
    if (i < ntiles) part_barrier<1, F::THREADS>();
  }

  part_barrier<2, F::HELP>();
  if (tq == 0) {  // the couples' sums over their tokens
    float2 dD = s.dD[tid], dbias = s.dbias[tid];
#pragma unroll
    for (int j = 1; j < F::STEP; ++j)
      dD = __fadd2_rn(dD, s.dD[tid + j * (F::DT / 2)]), dbias = __fadd2_rn(dbias, s.dbias[tid + j * (F::DT / 2)]);
    if (on0) part[DN + pd] = dD.x, part[DN + p.D + pd] = dbias.x;
    if (on1) part[DN + pd + 1] = dD.y, part[DN + p.D + pd + 1] = dbias.y;
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

// ------------------------------------------------------------------------------ host
// Enqueues the kernel and the sums of its partials; each type is compiled in a file of its own.
template <typename T>
int launch_bwd(Params p, void* dB, void* dC, float* dparams, cudaStream_t st, const char* who) {
  int rc = dispatch(p.N, [&](auto ln, auto npt) {
    using F = Bwd<decltype(ln)::value, decltype(npt)::value>;
    constexpr int LN = decltype(ln)::value, NPT = decltype(npt)::value;
    auto kernel = p.seq       ? p.couples ? scan_bwd_kernel<T, LN, NPT, true, true> : scan_bwd_kernel<T, LN, NPT, true, false>
                  : p.couples ? scan_bwd_kernel<T, LN, NPT, false, true>
                              : scan_bwd_kernel<T, LN, NPT, false, false>;
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
