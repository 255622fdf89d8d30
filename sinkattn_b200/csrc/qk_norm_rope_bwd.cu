// qk_norm_rope_bwd.cu — gradient of the hidden-wide Q/K norm + rotation
// (qk_norm_rope.cu), and the sum of partial rows that both norm gradients use.
//
// With g = the rotation transposed applied to the upstream gradient, u = g w
// and r = 1 / sqrt(mean x^2 + eps) over the hidden channels of a row:
//   dx = r (u - x r^2 mean(u x)),   dw = sum over rows of g x r.
// Memory-bound: x and the upstream gradient are read and dx written once
// (6 bf16 values per hidden channel of Q and K together). A team of 1, 2 or 4
// warps takes a row of Q or of K, at most 48 channels a lane, so that the row,
// its gradient and the lane's part of dw stay in registers and both sums of
// the row are reduced together.

#include <math.h>

#include "norm_rope.cuh"

namespace sa {
namespace nr {

__global__ void __launch_bounds__(256)
    partial_rows_kernel(const float* __restrict__ part, int rows, int cols, int pitch,
                        float* __restrict__ out0, float* __restrict__ out1, int cols0) {
  __shared__ float red[8][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), chain = threadIdx.x >> 5;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int r = chain; r < rows; r += 8) s += part[(int64_t)r * pitch + c];
  }
  red[chain][threadIdx.x & 31] = s;
  __syncthreads();
  if (chain == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x & 31];
    if (c < cols0) out0[c] = s; else out1[c - cols0] = s;
  }
}

int sum_partial_rows(const float* part, int rows, int cols, int pitch, float* out0, float* out1,
                     int cols0, cudaStream_t stream) {
  partial_rows_kernel<<<(cols + 31) / 32, 256, 0, stream>>>(part, rows, cols, pitch, out0, out1,
                                                            cols0);
  SA_CUDA_TRY(cudaGetLastError());
  return SA_OK;
}

}  // namespace nr

namespace qkrope_bwd {

using namespace sa::nr;

constexpr int kWarps = 4;
constexpr int kMaxHidden = 4096;

struct Params {
  const __nv_bfloat16* d[2];  // upstream gradients of q, k
  const __nv_bfloat16* x[2];
  __nv_bfloat16* o[2];
  const void* w[2];
  int64_t ds[2], xs[2], os[2];
  int rows, S, hidden, D;
  int w_dtype;
  float eps;
  const float *cos_t, *sin_t;
  int64_t fs;
  float* part;  // [partial rows][2][hidden], NULL without dw
};

// 8 channels of the upstream gradient, rotated back.
__device__ __forceinline__ void rotated(const Raw8<__nv_bfloat16>& raw, const float* cos_row,
                                        const float* sin_row, int c0, int D, float (&g)[8]) {
  unpack8(raw, g);
  if (cos_row == nullptr) return;
  const int p0 = (c0 % D) >> 1;
  const float4 c4 = __ldg(reinterpret_cast<const float4*>(cos_row + p0));
  const float4 s4 = __ldg(reinterpret_cast<const float4*>(sin_row + p0));
  const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float e = g[2 * i], o = g[2 * i + 1];
    g[2 * i] = e * c[i] + o * s[i];
    g[2 * i + 1] = o * c[i] - e * s[i];
  }
}

// W warps form a team that takes rows of one tensor: the block's teams are q,
// k, q, k (W = 1), q, k (W = 2) or one of them by the block's parity (W = 4).
template <int VPL, int W>
__global__ void __launch_bounds__(32 * kWarps) kernel(const Params p) {
  constexpr int kTeams = kWarps / W;
  __shared__ float2 sums[2][kWarps];
  extern __shared__ float stage[];  // W = 1: dw of the second q and k team
  const int team = (threadIdx.x >> 5) / W;
  const int64_t gteam = (int64_t)blockIdx.x * kTeams + team;
  const int which = (int)(gteam & 1);
  const int tl = threadIdx.x - team * 32 * W;  // thread of the team
  const int nvec = p.hidden >> 3;
  const float inv_n = 1.f / (float)p.hidden;
  float acc[VPL][8];
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  const int64_t step = (int64_t)gridDim.x * kTeams / 2;
  int turn = 0;
  for (int64_t row = gteam >> 1; row < p.rows; row += step, turn ^= 1) {
    const __nv_bfloat16* xr = p.x[which] + row * p.xs[which];
    const __nv_bfloat16* dr = p.d[which] + row * p.ds[which];
    __nv_bfloat16* orow = p.o[which] + row * p.os[which];
    Raw8<__nv_bfloat16> rx[VPL], rd[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int v = tl + i * 32 * W;
      rx[i] = rd[i] = Raw8<__nv_bfloat16>{};
      if (v < nvec) {
        rx[i] = load8(xr + v * 8);
        rd[i] = load8(dr + v * 8);
      }
    }
    const int s = (int)(row % p.S);
    const float* crow = p.cos_t != nullptr ? p.cos_t + (int64_t)s * p.fs : nullptr;
    const float* srow = p.sin_t != nullptr ? p.sin_t + (int64_t)s * p.fs : nullptr;
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int v = tl + i * 32 * W;
      if (v >= nvec) continue;
      float x[8], g[8], w[8];
      unpack8(rx[i], x);
      rotated(rd[i], crow, srow, v * 8, p.D, g);
      load_weight8(p.w[which], p.w_dtype, v * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fmaf(x[j], x[j], ss);
        dot = fmaf(g[j] * w[j], x[j], dot);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    if (W > 1) {
      // two buffers in turn: a warp writes the next row's sums only after the
      // whole team has passed this row's barrier
      if ((threadIdx.x & 31) == 0) sums[turn][threadIdx.x >> 5] = make_float2(ss, dot);
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(32 * W) : "memory");
      ss = dot = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        ss += sums[turn][team * W + w].x;
        dot += sums[turn][team * W + w].y;
      }
    }
    const float r = __fdiv_rn(1.f, __fsqrt_rn(ss * inv_n + p.eps));
    const float m = r * r * dot * inv_n;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int v = tl + i * 32 * W;
      if (v >= nvec) continue;
      float x[8], g[8], w[8];
      unpack8(rx[i], x);
      rotated(rd[i], crow, srow, v * 8, p.D, g);
      load_weight8(p.w[which], p.w_dtype, v * 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = fmaf(g[j] * r, x[j], acc[i][j]);
        x[j] = r * (g[j] * w[j] - x[j] * m);
      }
      store8(orow + v * 8, x);
    }
  }
  if (p.part == nullptr) return;
  if (W == 1) {
    if (team >= 2) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int v = tl + i * 32;
        if (v < nvec) store8(stage + which * p.hidden + v * 8, acc[i]);
      }
    }
    __syncthreads();
    if (team >= 2) return;
  }
  const int64_t prow = W == 4 ? blockIdx.x >> 1 : blockIdx.x;
  float* dst = p.part + (prow * 2 + which) * p.hidden;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int v = tl + i * 32 * W;
    if (v >= nvec) continue;
    if (W == 1) {
      const float* other = stage + which * p.hidden + v * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] += other[j];
    }
    store8(dst + v * 8, acc[i]);
  }
}

int max_blocks() { return sa::sm_count_current_device() * 4; }

}  // namespace qkrope_bwd
}  // namespace sa

extern "C" size_t sa_qk_norm_rope_bwd_workspace_size(int hidden) {
  if (hidden < 8) return 0;
  return (size_t)sa::qkrope_bwd::max_blocks() * 2 * hidden * sizeof(float);
}

extern "C" int sa_qk_norm_rope_bwd(const void* dq, const void* dk, int64_t dq_row_stride,
                                   int64_t dk_row_stride, const void* q, const void* k,
                                   int64_t q_row_stride, int64_t k_row_stride, int rows, int S,
                                   int hidden, int D, const void* w_q, const void* w_k,
                                   int w_is_bf16, float eps, const float* cos_table,
                                   const float* sin_table, int64_t freq_row_stride, void* dq_in,
                                   void* dk_in, int64_t dqi_row_stride, int64_t dki_row_stride,
                                   float* dw_q, float* dw_k, void* workspace, size_t ws_bytes,
                                   cudaStream_t stream) {
  using namespace sa::qkrope_bwd;
  const char* fn = "sa_qk_norm_rope_bwd";
  SA_CHECK_ARG(rows >= 0 && S >= 1 && D >= 8 && D % 8 == 0,
               "%s: bad sizes (D must be a multiple of 8)", fn);
  SA_CHECK_ARG(hidden >= 8 && hidden % 8 == 0 && hidden % D == 0 && hidden <= kMaxHidden,
               "%s: hidden (%d) must be a multiple of 8 and of D (%d), at most %d", fn, hidden, D,
               kMaxHidden);
  SA_CHECK_ARG((cos_table == nullptr) == (sin_table == nullptr),
               "%s: cos and sin tables go together", fn);
  SA_CHECK_ARG(cos_table == nullptr || (freq_row_stride >= D / 2 && freq_row_stride % 4 == 0 &&
                                        (((uintptr_t)cos_table | (uintptr_t)sin_table) & 15) == 0),
               "%s: frequency rows need D/2 entries, a stride that is a multiple of 4 and 16-byte "
               "aligned tables", fn);
  SA_CHECK_ARG(((dq_row_stride | dk_row_stride | q_row_stride | k_row_stride | dqi_row_stride |
                 dki_row_stride) & 7) == 0,
               "%s: row strides must be multiples of 8 elements", fn);
  SA_CHECK_ARG((((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)q | (uintptr_t)k | (uintptr_t)dq_in |
                 (uintptr_t)dk_in | (uintptr_t)w_q | (uintptr_t)w_k) & 15) == 0,
               "%s: tensors and weights must be 16-byte aligned", fn);
  SA_CHECK_ARG((w_q == nullptr) == (w_k == nullptr), "%s: weights go together", fn);
  SA_CHECK_ARG((dw_q == nullptr) == (dw_k == nullptr) && (dw_q == nullptr || w_q != nullptr),
               "%s: dw_q and dw_k go together and need weights", fn);
  const size_t need = dw_q != nullptr ? sa_qk_norm_rope_bwd_workspace_size(hidden) : 0;
  SA_CHECK_ARG(dw_q == nullptr || (workspace != nullptr && ws_bytes >= need &&
                                   (uintptr_t)workspace % 16 == 0),
               "%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", fn, need, ws_bytes);
  SA_CHECK_ARG(rows == 0 || (dq && dk && q && k && dq_in && dk_in), "%s: null tensor pointer", fn);
  int part_rows = 0;
  float* part = static_cast<float*>(workspace);
  if (rows > 0) {
    Params p;
    p.d[0] = static_cast<const __nv_bfloat16*>(dq); p.d[1] = static_cast<const __nv_bfloat16*>(dk);
    p.x[0] = static_cast<const __nv_bfloat16*>(q); p.x[1] = static_cast<const __nv_bfloat16*>(k);
    p.o[0] = static_cast<__nv_bfloat16*>(dq_in); p.o[1] = static_cast<__nv_bfloat16*>(dk_in);
    p.w[0] = w_q; p.w[1] = w_k;
    p.ds[0] = dq_row_stride; p.ds[1] = dk_row_stride;
    p.xs[0] = q_row_stride; p.xs[1] = k_row_stride;
    p.os[0] = dqi_row_stride; p.os[1] = dki_row_stride;
    p.rows = rows; p.S = S; p.hidden = hidden; p.D = D;
    p.w_dtype = w_is_bf16 ? SA_DTYPE_BF16 : SA_DTYPE_FP32;
    p.eps = eps;
    p.cos_t = cos_table; p.sin_t = sin_table; p.fs = freq_row_stride;
    p.part = dw_q != nullptr ? part : nullptr;
    // the narrowest team whose lanes hold at most 48 channels each
    const int W = hidden <= 1536 ? 1 : hidden <= 2 * 1536 ? 2 : 4;
    const int64_t rows_of_block = W == 1 ? 2 : 1;  // per tensor
    int64_t blocks = W == 4 ? 2 * (int64_t)rows : (rows + rows_of_block - 1) / rows_of_block;
    if (blocks > max_blocks()) blocks = max_blocks();  // even, as 4 blocks per SM
    part_rows = (int)(W == 4 ? blocks / 2 : blocks);
    const int vpl = (hidden / 8 + 32 * W - 1) / (32 * W);
    const size_t smem = W == 1 ? (size_t)2 * hidden * sizeof(float) : 0;
#define SA_LAUNCH(V, WW) kernel<V, WW><<<(int)blocks, 32 * kWarps, smem, stream>>>(p)
    if (W == 1) {
      if (vpl <= 2) SA_LAUNCH(2, 1);
      else if (vpl <= 4) SA_LAUNCH(4, 1);
      else SA_LAUNCH(6, 1);
    } else if (W == 2) {
      if (vpl <= 4) SA_LAUNCH(4, 2);
      else SA_LAUNCH(6, 2);
    } else {
      SA_LAUNCH(4, 4);
    }
#undef SA_LAUNCH
    SA_CUDA_TRY(cudaGetLastError());
  }
  if (dw_q == nullptr) return SA_OK;
  return sa::nr::sum_partial_rows(part, part_rows, 2 * hidden, 2 * hidden, dw_q, dw_k, hidden,
                                  stream);
}
