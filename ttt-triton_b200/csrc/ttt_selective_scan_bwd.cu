// Selective state space scan, backward: the entry points (the kernels are in
// selective_scan_bwd.cuh, compiled for each type in a file of its own), and the sums of
// partials in a fixed order.
#include "selective_scan.cuh"

namespace ttt {
namespace scan {

template <typename T>
int launch_bwd(Params p, void* dB, void* dC, float* dparams, cudaStream_t st, const char* who);

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
static int channels_of_a_cta(int N) { return 256 / shape_of(N).LN; }  // Bwd::DT

struct BwdScratch {
  size_t tiles, part_bc, part_p;  // bytes but for tiles
};
static BwdScratch bwd_scratch(int rows, int L, int D, int G, int N, int nchunks) {
  BwdScratch s;
  s.tiles = (D / G + channels_of_a_cta(N) - 1) / channels_of_a_cta(N);
  s.part_bc = s.tiles * rows * L * G * N * sizeof(float);
  s.part_p = (size_t)rows * nchunks * D * (N + 2) * sizeof(float);
  return s;
}

}  // namespace scan
}  // namespace ttt

using namespace ttt;

extern "C" size_t ttt_selective_scan_bwd_scratch_bytes(int rows, int L, int D, int G, int N) {
  if (rows < 1 || L < 1 || D < 1 || G < 1 || N < 1 || N > scan::kMaxStates || D % G) return 0;
  scan::Params p{};
  p.rows = rows, p.L = L, p.D = D, p.G = G, p.N = N;
  scan::plan_pieces(p, true);
  const scan::BwdScratch s = scan::bwd_scratch(rows, L, D, G, N, p.nchunks);
  return 2 * s.part_bc + s.part_p + scan::piece_bytes(p);
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
  scan::plan_pieces(p, true);
  const scan::BwdScratch s = scan::bwd_scratch(rows, L, D, G, N, p.nchunks);
  if ((rc = scan::plan_scratch(p, scratch, scratch_bytes, 2 * s.part_bc + s.part_p, who))) return rc;
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
