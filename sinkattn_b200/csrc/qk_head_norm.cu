// qk_head_norm.cu — RMSNorm of every query and key head over its own channels
// followed by the rotary embedding, and the gradient of both, each in one pass.
//
//   r = 1 / sqrt(mean_c x_c^2 + eps),  y_c = x_c r w_c,
//   (o_a, o_b) = (y_a cos - y_b sin, y_a sin + y_b cos) for the pairs
//   (a, b) = (2i, 2i+1) or (i, i + rot/2), i < rot/2; channels past rot are y.
// Gradient: with g = the rotation transposed applied to do and u = g w,
//   dx = r (u - x r^2 mean(u x)),  dw = sum over tokens and heads of g x r.
//
// Memory-bound: x read and o written once (the gradient reads do and x and
// writes dx). A lane holds 8 channels of a head, 16 lanes a head of 128, so
// the sums are shuffles inside a lane group, and a warp takes several heads of
// one token, whose angles and weights it loads once. Everything between the
// load and the store is fp32: the one rounding is that of the result.

#include <math.h>

#include "norm_rope.cuh"

namespace sa {
namespace headnorm {

using namespace sa::nr;

constexpr int kWarps = 4;    // warps of a block
constexpr int kUnroll = 4;   // heads of a lane group, loaded together

struct Params {
  const void *q, *k;
  int64_t qs0, qs1, qs2, ks0, ks1, ks2;
  void *qo, *ko;
  int64_t qos0, qos1, qos2, kos0, kos1, kos2;
  const void *dq, *dk;  // gradient only: upstream gradients
  int64_t dqs0, dqs1, dqs2, dks0, dks1, dks2;
  int B, S, Hq, Hk, D, rot;
  const void *wq, *wk;
  int w_dtype;
  float eps;
  const float *cos_t, *sin_t;
  int64_t fs;
  int table_rows;
  const void* pos;
  int pos_i64;
  int64_t ps0, ps1;
  int chunks;      // work items of a token
  int64_t items;   // tokens * chunks
  float* part;     // gradient only: per-block sums of dw [blocks][2][D]
  int32_t* status;
};

// cos and signed sin of this lane's 8 channels at its token: the rotated value
// is y cos + partner sin. SIGN is +1 for the rotation, -1 for its transpose.
template <bool INTER>
struct Angles {
  float c[INTER ? 4 : 8], s[INTER ? 4 : 8];
};

template <bool INTER>
__device__ __forceinline__ Angles<INTER> load_angles(const Params& p, int64_t row, int c0,
                                                     float sign) {
  Angles<INTER> a;
  constexpr int N = INTER ? 4 : 8;
  if (c0 < p.rot) {
    const int half = p.rot >> 1;
    const int i0 = INTER ? c0 >> 1 : (c0 < half ? c0 : c0 - half);
    const float m = INTER ? sign : (c0 < half ? -sign : sign);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t + row * p.fs + i0 + i));
      const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t + row * p.fs + i0 + i));
      a.c[i] = c4.x; a.c[i + 1] = c4.y; a.c[i + 2] = c4.z; a.c[i + 3] = c4.w;
      a.s[i] = m * s4.x; a.s[i + 1] = m * s4.y; a.s[i + 2] = m * s4.z; a.s[i + 3] = m * s4.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a.c[i] = 1.f;
      a.s[i] = 0.f;
    }
  }
  return a;
}

// Rotates 8 channels in place. Without interleaving the partner channels lie
// in another lane of the group (every lane of the warp takes part).
template <bool INTER>
__device__ __forceinline__ void rotate8(float (&y)[8], const Angles<INTER>& a, int partner) {
  if (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = y[2 * i], o = y[2 * i + 1];
      y[2 * i] = e * a.c[i] - o * a.s[i];
      y[2 * i + 1] = e * a.s[i] + o * a.c[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, y[i], partner);
      y[i] = y[i] * a.c[i] + other * a.s[i];
    }
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ int64_t table_row(const Params& p, int b, int s) {
  if (p.pos == nullptr) return s;
  const int64_t i = b * p.ps0 + s * p.ps1;
  return p.pos_i64 ? reinterpret_cast<const int64_t*>(p.pos)[i]
                   : (int64_t) reinterpret_cast<const int32_t*>(p.pos)[i];
}

// What a lane needs to know of its token.
struct Token {
  int b, s;
  int64_t row;  // of the tables
  bool bad;     // the position lies outside them
};

__device__ __forceinline__ Token token_of(const Params& p, int64_t t) {
  Token k;
  k.b = (int)(t / p.S);
  k.s = (int)(t - (int64_t)k.b * p.S);
  k.row = p.cos_t != nullptr ? table_row(p, k.b, k.s) : 0;
  k.bad = p.cos_t != nullptr && (k.row < 0 || k.row >= p.table_rows);
  if (k.bad) k.row = 0;
  return k;
}

// One warp per work item: kUnroll * (32 / G) heads of one token.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kWarps) fwd_kernel(const Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int64_t t = item / p.chunks;
  const int h0 = (int)(item - t * p.chunks) * (kUnroll * (32 / G)) + lane / G;
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  const Token tk = token_of(p, t);
  const int H = p.Hq + p.Hk;

  Raw8<T> raw[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int h = h0 + i * (32 / G);
    if (on && h < H) {
      const T* src = h < p.Hq
                         ? reinterpret_cast<const T*>(p.q) + tk.b * p.qs0 + tk.s * p.qs1 + h * p.qs2
                         : reinterpret_cast<const T*>(p.k) + tk.b * p.ks0 + tk.s * p.ks1 +
                               (h - p.Hq) * p.ks2;
      raw[i] = load8(src + c0);
    } else {
      raw[i] = Raw8<T>{};
    }
  }
  float wq[8], wk[8];
  load_weight8(p.wq, p.w_dtype, on ? c0 : 0, wq);
  load_weight8(p.wk, p.w_dtype, on ? c0 : 0, wk);
  const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, 1.f);
  const int partner = INTER || c0 >= p.rot ? lane : (c0 < p.rot / 2 ? lane + p.rot / 16
                                                                    : lane - p.rot / 16);
  if (tk.bad && lane == 0) report_status(p.status, SA_DEV_BAD_INDEX);
  const float inv_d = 1.f / (float)p.D;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int h = h0 + i * (32 / G);
    float x[8];
    unpack8(raw[i], x);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
    ss = group_sum<G>(ss);
    float r = __fdiv_rn(1.f, __fsqrt_rn(ss * inv_d + p.eps));
    if (tk.bad) r = __int_as_float(0x7fc00000);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (h < p.Hq ? wq[j] : wk[j]);
    rotate8<INTER>(x, ang, partner);
    if (on && h < H) {
      T* dst = h < p.Hq ? reinterpret_cast<T*>(p.qo) + tk.b * p.qos0 + tk.s * p.qos1 + h * p.qos2
                        : reinterpret_cast<T*>(p.ko) + tk.b * p.kos0 + tk.s * p.kos1 +
                              (h - p.Hq) * p.kos2;
      store8(dst + c0, x);
    }
  }
}

// Gradient: warps walk the work items with a stride of all warps, so that the
// sums of dw over a fixed set of tokens stay in registers; a block writes one
// partial row.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kWarps) bwd_kernel(const Params p) {
  __shared__ float red[kWarps][2][G * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  const int H = p.Hq + p.Hk;
  const int partner = INTER || c0 >= p.rot ? lane : (c0 < p.rot / 2 ? lane + p.rot / 16
                                                                    : lane - p.rot / 16);
  float wq[8], wk[8], aq[8], ak[8];
  load_weight8(p.wq, p.w_dtype, on ? c0 : 0, wq);
  load_weight8(p.wk, p.w_dtype, on ? c0 : 0, wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) aq[j] = ak[j] = 0.f;
  const float inv_d = 1.f / (float)p.D;
  const int64_t step = (int64_t)gridDim.x * kWarps;
  for (int64_t item = (int64_t)blockIdx.x * kWarps + warp; item < p.items; item += step) {
    const int64_t t = item / p.chunks;
    const int h0 = (int)(item - t * p.chunks) * (kUnroll * (32 / G)) + lane / G;
    const Token tk = token_of(p, t);
    Raw8<T> rx[kUnroll], rd[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int h = h0 + i * (32 / G);
      rx[i] = rd[i] = Raw8<T>{};
      if (on && h < H) {
        const bool is_q = h < p.Hq;
        const int hh = is_q ? h : h - p.Hq;
        rx[i] = load8((is_q ? reinterpret_cast<const T*>(p.q) + tk.b * p.qs0 + tk.s * p.qs1 +
                                  hh * p.qs2
                            : reinterpret_cast<const T*>(p.k) + tk.b * p.ks0 + tk.s * p.ks1 +
                                  hh * p.ks2) + c0);
        rd[i] = load8((is_q ? reinterpret_cast<const T*>(p.dq) + tk.b * p.dqs0 + tk.s * p.dqs1 +
                                  hh * p.dqs2
                            : reinterpret_cast<const T*>(p.dk) + tk.b * p.dks0 + tk.s * p.dks1 +
                                  hh * p.dks2) + c0);
      }
    }
    const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, -1.f);
    if (tk.bad && lane == 0) report_status(p.status, SA_DEV_BAD_INDEX);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int h = h0 + i * (32 / G);
      const bool is_q = h < p.Hq;
      float x[8], g[8];
      unpack8(rx[i], x);
      unpack8(rd[i], g);
      rotate8<INTER>(g, ang, partner);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fmaf(x[j], x[j], ss);
        dot = fmaf(g[j] * (is_q ? wq[j] : wk[j]), x[j], dot);
      }
      ss = group_sum<G>(ss);
      dot = group_sum<G>(dot);
      float r = __fdiv_rn(1.f, __fsqrt_rn(ss * inv_d + p.eps));
      if (tk.bad) r = __int_as_float(0x7fc00000);
      const float m = r * r * dot * inv_d;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j] = r * (g[j] * (is_q ? wq[j] : wk[j]) - x[j] * m);
        const float a = g[j] * x[j] * r;  // 0 for heads past H: their g and x are 0
        if (h < H) {
          if (is_q) aq[j] += a; else ak[j] += a;
        }
      }
      if (on && h < H) {
        const int hh = is_q ? h : h - p.Hq;
        T* dst = is_q ? reinterpret_cast<T*>(p.qo) + tk.b * p.qos0 + tk.s * p.qos1 + hh * p.qos2
                      : reinterpret_cast<T*>(p.ko) + tk.b * p.kos0 + tk.s * p.kos1 + hh * p.kos2;
        store8(dst + c0, o);
      }
    }
  }
  if (p.part == nullptr) return;
  // the warp's lane groups hold sums of the same channels
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o >= G; o >>= 1) {
      aq[j] += __shfl_xor_sync(0xffffffffu, aq[j], o);
      ak[j] += __shfl_xor_sync(0xffffffffu, ak[j], o);
    }
    if (lane < G) {
      red[warp][0][c0 + j] = aq[j];
      red[warp][1][c0 + j] = ak[j];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.D; c += 32 * kWarps) {
    const int which = c >= p.D, cc = which ? c - p.D : c;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w][which][cc];
    p.part[(int64_t)blockIdx.x * 2 * p.D + c] = s;
  }
}

template <typename T, int G>
void launch_g(const Params& p, bool inter, bool bwd, int grid, cudaStream_t stream) {
  if (bwd) {
    if (inter) bwd_kernel<T, G, true><<<grid, 32 * kWarps, 0, stream>>>(p);
    else bwd_kernel<T, G, false><<<grid, 32 * kWarps, 0, stream>>>(p);
  } else {
    if (inter) fwd_kernel<T, G, true><<<grid, 32 * kWarps, 0, stream>>>(p);
    else fwd_kernel<T, G, false><<<grid, 32 * kWarps, 0, stream>>>(p);
  }
}

// lanes of a head: the power of two that covers D / 8, at least 4
int group_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

template <typename T>
void launch_t(const Params& p, bool inter, bool bwd, int grid, cudaStream_t stream) {
  switch (group_of(p.D)) {
    case 4: launch_g<T, 4>(p, inter, bwd, grid, stream); break;
    case 8: launch_g<T, 8>(p, inter, bwd, grid, stream); break;
    case 16: launch_g<T, 16>(p, inter, bwd, grid, stream); break;
    default: launch_g<T, 32>(p, inter, bwd, grid, stream); break;
  }
}

int dispatch(const Params& p, int dtype, bool inter, bool bwd, int grid, cudaStream_t stream) {
  if (dtype == SA_DTYPE_BF16) launch_t<__nv_bfloat16>(p, inter, bwd, grid, stream);
  else if (dtype == SA_DTYPE_FP16) launch_t<__half>(p, inter, bwd, grid, stream);
  else launch_t<float>(p, inter, bwd, grid, stream);
  SA_CUDA_TRY(cudaGetLastError());
  return SA_OK;
}

bool aligned_ok(const void* base, const int64_t st[4], int dtype) {
  if (base == nullptr) return true;
  const int64_t mult = dtype == SA_DTYPE_FP32 ? 4 : 8;
  return (uintptr_t)base % 16 == 0 && st != nullptr && st[3] == 1 && st[0] >= 0 && st[1] >= 0 &&
         st[2] >= 0 && st[0] % mult == 0 && st[1] % mult == 0 && st[2] % mult == 0;
}

// Arguments that the forward and the gradient share.
int check(const char* fn, int B, int S, int Hq, int Hk, int D, int dtype, const void* w_q,
          const void* w_k, int w_dtype, const float* cos_t, const float* sin_t, int64_t fs,
          int table_rows, int rot, int interleaved, const void* positions,
          const int64_t pos_strides[2]) {
  SA_CHECK_ARG(B >= 0 && S >= 0 && Hq >= 1 && Hk >= 0, "%s: bad sizes (B %d, S %d, Hq %d, Hk %d)",
               fn, B, S, Hq, Hk);
  SA_CHECK_ARG((int64_t)B * S <= 0x7fffffff && Hq <= 65536 && Hk <= 65536,
               "%s: too many tokens or heads", fn);
  SA_CHECK_ARG(D >= 8 && D <= 256 && D % 8 == 0, "%s: head dim must be a multiple of 8 up to 256, "
               "got %d", fn, D);
  SA_CHECK_ARG(dtype >= SA_DTYPE_BF16 && dtype <= SA_DTYPE_FP32 && w_dtype >= SA_DTYPE_BF16 &&
                   w_dtype <= SA_DTYPE_FP32, "%s: unknown dtype", fn);
  SA_CHECK_ARG((w_q == nullptr) == (w_k == nullptr) || Hk == 0, "%s: weights go together", fn);
  SA_CHECK_ARG((((uintptr_t)w_q | (uintptr_t)w_k) & 15) == 0,
               "%s: weights must be 16-byte aligned", fn);
  SA_CHECK_ARG((cos_t == nullptr) == (sin_t == nullptr), "%s: cos and sin tables go together", fn);
  if (cos_t != nullptr) {
    SA_CHECK_ARG(rot >= 8 && rot <= D && rot % (interleaved ? 8 : 16) == 0,
                 "%s: the rotated channels must be a multiple of %d up to D, got %d", fn,
                 interleaved ? 8 : 16, rot);
    SA_CHECK_ARG(fs >= rot / 2 && fs % 4 == 0 &&
                     (((uintptr_t)cos_t | (uintptr_t)sin_t) & 15) == 0,
                 "%s: table rows need a stride that is a multiple of 4 and 16-byte aligned tables",
                 fn);
    SA_CHECK_ARG(table_rows >= 1 && (positions != nullptr || table_rows >= S),
                 "%s: %d table rows for %d tokens", fn, table_rows, S);
  }
  SA_CHECK_ARG(positions == nullptr || (cos_t != nullptr && pos_strides != nullptr),
               "%s: positions need tables and strides", fn);
  return SA_OK;
}

void common(Params& p, const void* q, const void* k, const int64_t* qs, const int64_t* ks, int B,
            int S, int Hq, int Hk, int D, const void* w_q, const void* w_k, int w_dtype, float eps,
            const float* cos_t, const float* sin_t, int64_t fs, int table_rows, int rot,
            const void* positions, int pos_i64, const int64_t* pos_strides, void* qo, void* ko,
            const int64_t* qos, const int64_t* kos, int32_t* status) {
  static const int64_t zero[4] = {0, 0, 0, 1};
  if (Hk == 0) ks = kos = zero;
  p = Params{};
  p.q = q; p.k = k; p.qo = qo; p.ko = ko;
  p.qs0 = qs[0]; p.qs1 = qs[1]; p.qs2 = qs[2];
  p.ks0 = ks[0]; p.ks1 = ks[1]; p.ks2 = ks[2];
  p.qos0 = qos[0]; p.qos1 = qos[1]; p.qos2 = qos[2];
  p.kos0 = kos[0]; p.kos1 = kos[1]; p.kos2 = kos[2];
  p.B = B; p.S = S; p.Hq = Hq; p.Hk = Hk; p.D = D;
  p.rot = cos_t != nullptr ? rot : 0;
  p.wq = w_q; p.wk = w_k; p.w_dtype = w_dtype; p.eps = eps;
  p.cos_t = cos_t; p.sin_t = sin_t; p.fs = fs; p.table_rows = table_rows;
  p.pos = positions; p.pos_i64 = pos_i64;
  if (positions != nullptr) { p.ps0 = pos_strides[0]; p.ps1 = pos_strides[1]; }
  const int per = kUnroll * (32 / group_of(D));
  p.chunks = (Hq + Hk + per - 1) / per;
  p.items = (int64_t)B * S * p.chunks;
  p.status = status;
}

// Blocks of the gradient kernel: enough to fill the GPU, each a partial row.
int bwd_blocks(int64_t items) {
  const int64_t want = (items + kWarps - 1) / kWarps;
  const int64_t most = (int64_t)sa::sm_count_current_device() * 4;
  return (int)(want < most ? want : most);
}

}  // namespace headnorm
}  // namespace sa

extern "C" int sa_qk_head_norm_rope(
    const void* q, const void* k, const int64_t q_strides[4], const int64_t k_strides[4], int B,
    int S, int Hq, int Hk, int D, int dtype, const void* w_q, const void* w_k, int w_dtype,
    float eps, const float* cos_table, const float* sin_table, int64_t freq_row_stride,
    int table_rows, int rot_dim, int interleaved, const void* positions, int positions_i64,
    const int64_t pos_strides[2], void* q_out, void* k_out, const int64_t qo_strides[4],
    const int64_t ko_strides[4], int32_t* status, cudaStream_t stream) {
  using namespace sa::headnorm;
  const char* fn = "sa_qk_head_norm_rope";
  int rc = check(fn, B, S, Hq, Hk, D, dtype, w_q, w_k, w_dtype, cos_table, sin_table,
                 freq_row_stride, table_rows, rot_dim, interleaved, positions, pos_strides);
  if (rc != SA_OK) return rc;
  if (B == 0 || S == 0) return SA_OK;
  SA_CHECK_ARG(q && q_out && (Hk == 0 || (k && k_out)), "%s: null tensor pointer", fn);
  SA_CHECK_ARG(aligned_ok(q, q_strides, dtype) && aligned_ok(q_out, qo_strides, dtype) &&
                   (Hk == 0 || (aligned_ok(k, k_strides, dtype) &&
                                aligned_ok(k_out, ko_strides, dtype))),
               "%s: tensors need stride(dim)=1, 16-byte aligned bases and strides", fn);
  Params p;
  common(p, q, k, q_strides, k_strides, B, S, Hq, Hk, D, w_q, w_k, w_dtype, eps, cos_table,
         sin_table, freq_row_stride, table_rows, rot_dim, positions, positions_i64, pos_strides,
         q_out, k_out, qo_strides, ko_strides, status);
  const int64_t blocks = (p.items + kWarps - 1) / kWarps;
  SA_CHECK_ARG(blocks <= 0x7fffffff, "%s: too many tokens", fn);
  return dispatch(p, dtype, interleaved != 0, false, (int)blocks, stream);
}

extern "C" size_t sa_qk_head_norm_rope_bwd_workspace_size(int D) {
  if (D < 8) return 0;
  return (size_t)sa::sm_count_current_device() * 4 * 2 * D * sizeof(float);
}

extern "C" int sa_qk_head_norm_rope_bwd(
    const void* dq, const void* dk, const int64_t dq_strides[4], const int64_t dk_strides[4],
    const void* q, const void* k, const int64_t q_strides[4], const int64_t k_strides[4], int B,
    int S, int Hq, int Hk, int D, int dtype, const void* w_q, const void* w_k, int w_dtype,
    float eps, const float* cos_table, const float* sin_table, int64_t freq_row_stride,
    int table_rows, int rot_dim, int interleaved, const void* positions, int positions_i64,
    const int64_t pos_strides[2], void* dq_in, void* dk_in, const int64_t dqi_strides[4],
    const int64_t dki_strides[4], float* dw_q, float* dw_k, void* workspace, size_t ws_bytes,
    int32_t* status, cudaStream_t stream) {
  using namespace sa::headnorm;
  const char* fn = "sa_qk_head_norm_rope_bwd";
  int rc = check(fn, B, S, Hq, Hk, D, dtype, w_q, w_k, w_dtype, cos_table, sin_table,
                 freq_row_stride, table_rows, rot_dim, interleaved, positions, pos_strides);
  if (rc != SA_OK) return rc;
  const bool weights = dw_q != nullptr || dw_k != nullptr;
  SA_CHECK_ARG(!weights || (w_q != nullptr && dw_q != nullptr && (Hk == 0 || dw_k != nullptr)),
               "%s: dw_q and dw_k go together and need weights", fn);
  const size_t need = weights ? sa_qk_head_norm_rope_bwd_workspace_size(D) : 0;
  SA_CHECK_ARG(!weights || (workspace != nullptr && ws_bytes >= need &&
                            (uintptr_t)workspace % 16 == 0),
               "%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", fn, need, ws_bytes);
  int blocks = 0;
  float* part = static_cast<float*>(workspace);
  if (B > 0 && S > 0) {
    SA_CHECK_ARG(dq && q && dq_in && (Hk == 0 || (dk && k && dk_in)), "%s: null tensor pointer",
                 fn);
    SA_CHECK_ARG(aligned_ok(q, q_strides, dtype) && aligned_ok(dq, dq_strides, dtype) &&
                     aligned_ok(dq_in, dqi_strides, dtype) &&
                     (Hk == 0 || (aligned_ok(k, k_strides, dtype) &&
                                  aligned_ok(dk, dk_strides, dtype) &&
                                  aligned_ok(dk_in, dki_strides, dtype))),
                 "%s: tensors need stride(dim)=1, 16-byte aligned bases and strides", fn);
    Params p;
    common(p, q, k, q_strides, k_strides, B, S, Hq, Hk, D, w_q, w_k, w_dtype, eps, cos_table,
           sin_table, freq_row_stride, table_rows, rot_dim, positions, positions_i64, pos_strides,
           dq_in, dk_in, dqi_strides, dki_strides, status);
    p.dq = dq; p.dk = dk;
    p.dqs0 = dq_strides[0]; p.dqs1 = dq_strides[1]; p.dqs2 = dq_strides[2];
    if (Hk > 0) { p.dks0 = dk_strides[0]; p.dks1 = dk_strides[1]; p.dks2 = dk_strides[2]; }
    p.part = weights ? part : nullptr;
    blocks = bwd_blocks(p.items);
    rc = dispatch(p, dtype, interleaved != 0, true, blocks, stream);
    if (rc != SA_OK) return rc;
  }
  if (!weights) return SA_OK;
  return sa::nr::sum_partial_rows(part, blocks, Hk > 0 ? 2 * D : D, 2 * D, dw_q, dw_k, D, stream);
}
