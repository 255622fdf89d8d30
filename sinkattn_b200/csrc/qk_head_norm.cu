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
// writes dx). A lane holds 8 channels of a head (16 lanes a head of 128), so
// the sums are shuffles inside a lane group. A warp takes 4 heads per lane
// group of one token and one tensor, all loaded before the first is used, and
// folds weight, cosine and sine into the two factors of each channel once for
// all of them; the arithmetic is f32x2, as the scalar form was bound by its
// instructions. Everything between the load and the store is fp32: the one
// rounding is that of the result.

#include <math.h>

#include "norm_rope.cuh"

namespace sa {
namespace headnorm {

using namespace sa::nr;

constexpr int kUnroll = 4;   // heads of a lane group, loaded together
constexpr int kUnrollBwd = 2;  // as many vectors: two tensors are read
constexpr int kMaxWarps = 8; // warps of a block: the chunks of one token
constexpr int kMaxHeads = 8192;  // of q and k together
constexpr int kMaxRows = (kMaxHeads / kUnrollBwd + 2) / kMaxWarps + 1;  // blocks of one token

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
  int chunks_q, chunks;  // warps of a token: those of q, then those of k
  int tokens;
  float* part;     // gradient only: per-block sums of dw [blocks][2][D]
  int32_t* status;
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a warp needs to know of its token.
struct Token {
  int b, s;
  int64_t row;  // of the tables
  bool bad;     // the position lies outside them
};

__device__ __forceinline__ Token token_of(const Params& p, int t) {
  Token k;
  k.b = (int)((unsigned)t / (unsigned)p.S);
  k.s = t - k.b * p.S;
  k.row = k.s;
  if (p.pos != nullptr) {
    const int64_t i = k.b * p.ps0 + k.s * p.ps1;
    k.row = p.pos_i64 ? reinterpret_cast<const int64_t*>(p.pos)[i]
                      : (int64_t) reinterpret_cast<const int32_t*>(p.pos)[i];
  }
  k.bad = p.cos_t != nullptr && (k.row < 0 || k.row >= p.table_rows);
  if (k.bad) k.row = 0;
  return k;
}

// Cosine and sine of a lane's 8 channels: one pair per two channels with
// interleaving (c[0], c[1] for channels 0-3, 4-7 as pairs), else one per
// channel in planar order, the sine signed so that out = y c + partner s.
template <bool INTER>
struct Angles {
  uint64_t c[INTER ? 2 : 4], s[INTER ? 2 : 4];
};

// sign: +1 for the rotation, -1 for its transpose.
template <bool INTER>
__device__ __forceinline__ Angles<INTER> load_angles(const Params& p, int64_t row, int c0,
                                                     float sign) {
  Angles<INTER> a;
  if (INTER) {
    float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c0 < p.rot) {
      c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t + row * p.fs + (c0 >> 1)));
      s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t + row * p.fs + (c0 >> 1)));
    }
    a.c[0] = f2_pack(c4.x, c4.y); a.c[1] = f2_pack(c4.z, c4.w);
    a.s[0] = f2_pack(sign * s4.x, sign * s4.y); a.s[1] = f2_pack(sign * s4.z, sign * s4.w);
  } else {
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { c[i] = 1.f; s[i] = 0.f; }
    if (c0 < p.rot) {
      const int half = p.rot >> 1;
      const int i0 = c0 < half ? c0 : c0 - half;
      const float m = c0 < half ? -sign : sign;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t + row * p.fs + i0 + i));
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t + row * p.fs + i0 + i));
        c[i] = c4.x; c[i + 1] = c4.y; c[i + 2] = c4.z; c[i + 3] = c4.w;
        s[i] = m * s4.x; s[i + 1] = m * s4.y; s[i + 2] = m * s4.z; s[i + 3] = m * s4.w;
      }
    }
    const V8 cp = planar(c), sp = planar(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a.c[i] = cp.v[i];
      a.s[i] = sp.v[i];
    }
  }
  return a;
}

// The lane that holds the other channels of a lane's pairs (itself when they
// are its own) and the channels it holds.
template <bool INTER>
__device__ __forceinline__ int partner_of(const Params& p, int lane, int c0, int& pc0) {
  pc0 = c0;
  if (INTER || c0 >= p.rot) return lane;
  const int half = p.rot >> 1, d = c0 < half ? half : -half;
  pc0 = c0 + d;
  return lane + d / 8;
}

// This warp's heads: tensor (0 q, 1 k), the first head of its lane group and
// the number of heads of the tensor.
struct Heads {
  int which, h0, H;
};

template <int G, int U>
__device__ __forceinline__ Heads heads_of(const Params& p, int chunk, int lane) {
  Heads h;
  h.which = chunk >= p.chunks_q ? 1 : 0;
  h.H = h.which ? p.Hk : p.Hq;
  h.h0 = (h.which ? chunk - p.chunks_q : chunk) * (U * (32 / G)) + lane / G;
  return h;
}

// One warp per token and chunk of heads.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kMaxWarps, INTER ? 4 : 3) fwd_kernel(const Params p) {
  const int lane = threadIdx.x & 31;
  const int chunk = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (chunk >= p.chunks) return;
  const Heads hd = heads_of<G, kUnroll>(p, chunk, lane);
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  const Token tk = token_of(p, blockIdx.x);
  const T* src = hd.which
                     ? reinterpret_cast<const T*>(p.k) + tk.b * p.ks0 + tk.s * p.ks1 + c0
                     : reinterpret_cast<const T*>(p.q) + tk.b * p.qs0 + tk.s * p.qs1 + c0;
  T* dst = hd.which ? reinterpret_cast<T*>(p.ko) + tk.b * p.kos0 + tk.s * p.kos1 + c0
                    : reinterpret_cast<T*>(p.qo) + tk.b * p.qos0 + tk.s * p.qos1 + c0;
  const int64_t hs = hd.which ? p.ks2 : p.qs2, ohs = hd.which ? p.kos2 : p.qos2;
  Raw8<T> raw[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int h = hd.h0 + i * (32 / G);
    raw[i] = Raw8<T>{};
    if (on && h < hd.H) raw[i] = load8(src + h * hs);
  }
  int pc0;
  const int partner = partner_of<INTER>(p, lane, c0, pc0);
  const void* wp = hd.which ? p.wk : p.wq;
  const V8 w = load_weight8(wp, p.w_dtype, on ? c0 : 0);
  const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, 1.f);
  // out = r (x a + other b) per channel, other = the pair's second channel
  V8 a, b;
  if (INTER) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t minus = f2_pack(-1.f, -1.f);
      a.v[2 * i] = f2_mul(w.v[2 * i], ang.c[i]);
      b.v[2 * i] = f2_mul(f2_mul(w.v[2 * i + 1], ang.s[i]), minus);
      a.v[2 * i + 1] = f2_mul(w.v[2 * i + 1], ang.c[i]);
      b.v[2 * i + 1] = f2_mul(w.v[2 * i], ang.s[i]);
    }
  } else {
    const V8 wo = load_weight8(wp, p.w_dtype, on ? pc0 : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a.v[i] = f2_mul(w.v[i], ang.c[i]);
      b.v[i] = f2_mul(wo.v[i], ang.s[i]);
    }
  }
  if (tk.bad && lane == 0) report_status(p.status, SA_DEV_BAD_INDEX);
  const float inv_d = 1.f / (float)p.D;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int h = hd.h0 + i * (32 / G);
    const V8 x = unpack8(raw[i]);
    uint64_t s2 = f2_mul(x.v[0], x.v[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) s2 = f2_fma(x.v[j], x.v[j], s2);
    const float ss = group_sum<G>(sum2(s2));
    float r = inv_sqrt(fmaf(ss, inv_d, p.eps));
    if (tk.bad) r = __int_as_float(0x7fc00000);
    const uint64_t r2 = f2_pack(r, r);
    V8 other;
    if (INTER) {
      other = V8{{x.v[1], x.v[0], x.v[3], x.v[2]}};
    } else {
      other = unpack8(shfl8(raw[i], partner));
    }
    V8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o.v[j] = f2_mul(f2_fma(x.v[j], a.v[j], f2_mul(other.v[j], b.v[j])), r2);
    if (on && h < hd.H) store8(dst + h * ohs, o);
  }
}

// Gradient: a warp keeps its chunk of heads and walks the tokens with a stride
// of the grid, so that its part of dw stays in registers; a block writes one
// partial row.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kMaxWarps, sizeof(T) == 2 ? 3 : 2) bwd_kernel(const Params p) {
  __shared__ float red[kMaxWarps][G * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int chunk = blockIdx.y * warps + warp;
  const Heads hd = heads_of<G, kUnrollBwd>(p, chunk, lane);
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  int pc0;
  const int partner = partner_of<INTER>(p, lane, c0, pc0);
  const V8 w = load_weight8(hd.which ? p.wk : p.wq, p.w_dtype, on ? c0 : 0);
  const T* xb = reinterpret_cast<const T*>(hd.which ? p.k : p.q) + c0;
  const T* db = reinterpret_cast<const T*>(hd.which ? p.dk : p.dq) + c0;
  T* ob = reinterpret_cast<T*>(hd.which ? p.ko : p.qo) + c0;
  const int64_t xs0 = hd.which ? p.ks0 : p.qs0, xs1 = hd.which ? p.ks1 : p.qs1,
                xs2 = hd.which ? p.ks2 : p.qs2;
  const int64_t ds0 = hd.which ? p.dks0 : p.dqs0, ds1 = hd.which ? p.dks1 : p.dqs1,
                ds2 = hd.which ? p.dks2 : p.dqs2;
  const int64_t os0 = hd.which ? p.kos0 : p.qos0, os1 = hd.which ? p.kos1 : p.qos1,
                os2 = hd.which ? p.kos2 : p.qos2;
  release_next_kernel();
  V8 acc = fill8(0.f);
  const float inv_d = 1.f / (float)p.D;
  if (chunk < p.chunks) {
    for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
      const Token tk = token_of(p, t);
      const T* xt = xb + tk.b * xs0 + tk.s * xs1;
      const T* dt = db + tk.b * ds0 + tk.s * ds1;
      T* ot = ob + tk.b * os0 + tk.s * os1;
      Raw8<T> rx[kUnrollBwd], rd[kUnrollBwd];
#pragma unroll
      for (int i = 0; i < kUnrollBwd; ++i) {
        const int h = hd.h0 + i * (32 / G);
        rx[i] = rd[i] = Raw8<T>{};
        if (on && h < hd.H) {
          rx[i] = load8(xt + h * xs2);
          rd[i] = load8(dt + h * ds2);
        }
      }
      const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, -1.f);
      const uint64_t minus = f2_pack(-1.f, -1.f);
      const uint64_t pos_s[2] = {f2_mul(ang.s[0], minus), f2_mul(ang.s[1], minus)};
      if (tk.bad && lane == 0) report_status(p.status, SA_DEV_BAD_INDEX);
#pragma unroll
      for (int i = 0; i < kUnrollBwd; ++i) {
        const int h = hd.h0 + i * (32 / G);
        const V8 x = unpack8(rx[i]), d = unpack8(rd[i]);
        V8 g;
        if (INTER) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // the sine comes negated: g_e = d_e c + d_o s, g_o = d_o c - d_e s
            g.v[2 * j] = f2_fma(d.v[2 * j], ang.c[j], f2_mul(d.v[2 * j + 1], pos_s[j]));
            g.v[2 * j + 1] = f2_fma(d.v[2 * j + 1], ang.c[j], f2_mul(d.v[2 * j], ang.s[j]));
          }
        } else {
          const V8 other = unpack8(shfl8(rd[i], partner));
#pragma unroll
          for (int j = 0; j < 4; ++j)
            g.v[j] = f2_fma(d.v[j], ang.c[j], f2_mul(other.v[j], ang.s[j]));
        }
        V8 u;
        uint64_t s2 = f2_mul(x.v[0], x.v[0]);
        u.v[0] = f2_mul(g.v[0], w.v[0]);
        uint64_t t2 = f2_mul(u.v[0], x.v[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) {
          s2 = f2_fma(x.v[j], x.v[j], s2);
          u.v[j] = f2_mul(g.v[j], w.v[j]);
          t2 = f2_fma(u.v[j], x.v[j], t2);
        }
        const float ss = group_sum<G>(sum2(s2)), dot = group_sum<G>(sum2(t2));
        float r = inv_sqrt(fmaf(ss, inv_d, p.eps));
        if (tk.bad) r = __int_as_float(0x7fc00000);
        const float m = -r * r * r * dot * inv_d;
        const uint64_t r2 = f2_pack(r, r), m2 = f2_pack(m, m);
        if (on && h < hd.H) {
          V8 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc.v[j] = f2_fma(f2_mul(g.v[j], r2), x.v[j], acc.v[j]);
            o.v[j] = f2_fma(x.v[j], m2, f2_mul(u.v[j], r2));
          }
          store8(ot + h * os2, o);
        }
      }
    }
  }
  if (p.part == nullptr) return;
  // the warp's lane groups hold sums of the same channels
  float a8[8];
  channels(acc, a8);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o >= G; o >>= 1) a8[j] += __shfl_xor_sync(0xffffffffu, a8[j], o);
    if (lane < G) red[warp][c0 + j] = a8[j];
  }
  __syncthreads();
  float* row = p.part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.D;
  const int first_k = p.chunks_q - blockIdx.y * warps;  // the first warp on k
  for (int c = threadIdx.x; c < 2 * p.D; c += blockDim.x) {
    const int which = c >= p.D, cc = which ? c - p.D : c;
    float s = 0.f;
    for (int v = 0; v < warps; ++v)
      if ((v >= first_k) == (which != 0)) s += red[v][cc];
    row[c] = s;
  }
}

template <typename T, int G>
void launch_g(const Params& p, bool inter, bool bwd, dim3 grid, int threads,
              cudaStream_t stream) {
  if (bwd) {
    if (inter) bwd_kernel<T, G, true><<<grid, threads, 0, stream>>>(p);
    else bwd_kernel<T, G, false><<<grid, threads, 0, stream>>>(p);
  } else {
    if (inter) fwd_kernel<T, G, true><<<grid, threads, 0, stream>>>(p);
    else fwd_kernel<T, G, false><<<grid, threads, 0, stream>>>(p);
  }
}

// lanes of a head: the power of two that covers D / 8, at least 4
int group_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

template <typename T>
void launch_t(const Params& p, bool inter, bool bwd, dim3 grid, int threads,
              cudaStream_t stream) {
  switch (group_of(p.D)) {
    case 4: launch_g<T, 4>(p, inter, bwd, grid, threads, stream); break;
    case 8: launch_g<T, 8>(p, inter, bwd, grid, threads, stream); break;
    case 16: launch_g<T, 16>(p, inter, bwd, grid, threads, stream); break;
    default: launch_g<T, 32>(p, inter, bwd, grid, threads, stream); break;
  }
}

int dispatch(const Params& p, int dtype, bool inter, bool bwd, dim3 grid, int threads,
             cudaStream_t stream) {
  if (dtype == SA_DTYPE_BF16) launch_t<__nv_bfloat16>(p, inter, bwd, grid, threads, stream);
  else if (dtype == SA_DTYPE_FP16) launch_t<__half>(p, inter, bwd, grid, threads, stream);
  else launch_t<float>(p, inter, bwd, grid, threads, stream);
  SA_CUDA_TRY(cudaGetLastError());
  return SA_OK;
}

// Blocks take the chunks of one token, split evenly over as few as possible.
void shape(const Params& p, int& warps, int& rows) {
  rows = (p.chunks + kMaxWarps - 1) / kMaxWarps;
  warps = (p.chunks + rows - 1) / rows;
}

// Tokens in flight of the gradient kernel (grid.x): 24 warps per SM, a
// partial row of dw from each block.
constexpr int kBwdWarpsPerSm = 24;
int bwd_grid(int tokens, int warps, int rows) {
  const int64_t most =
      ((int64_t)sa::sm_count_current_device() * kBwdWarpsPerSm + warps * rows - 1) / (warps * rows);
  return (int)(tokens < most ? tokens : most);
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
  SA_CHECK_ARG((int64_t)B * S <= 0x7fffffff && Hq + Hk <= kMaxHeads,
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
            const int64_t* qos, const int64_t* kos, int unroll, int32_t* status) {
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
  const int per = unroll * (32 / group_of(D));
  p.chunks_q = (Hq + per - 1) / per;
  p.chunks = p.chunks_q + (Hk + per - 1) / per;
  p.tokens = B * S;
  p.status = status;
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
         q_out, k_out, qo_strides, ko_strides, kUnroll, status);
  int warps, rows;
  shape(p, warps, rows);
  return dispatch(p, dtype, interleaved != 0, false, dim3((unsigned)p.tokens, (unsigned)rows),
                  32 * warps, stream);
}

extern "C" size_t sa_qk_head_norm_rope_bwd_workspace_size(int D) {
  if (D < 8) return 0;
  // at most kBwdWarpsPerSm blocks (of one warp) per SM, or one per block row
  return (size_t)(sa::sm_count_current_device() * sa::headnorm::kBwdWarpsPerSm +
                  sa::headnorm::kMaxRows) * 2 * D * sizeof(float);
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
           dq_in, dk_in, dqi_strides, dki_strides, kUnrollBwd, status);
    p.dq = dq; p.dk = dk;
    p.dqs0 = dq_strides[0]; p.dqs1 = dq_strides[1]; p.dqs2 = dq_strides[2];
    if (Hk > 0) { p.dks0 = dk_strides[0]; p.dks1 = dk_strides[1]; p.dks2 = dk_strides[2]; }
    p.part = weights ? part : nullptr;
    int warps, rows;
    shape(p, warps, rows);
    const int gx = bwd_grid(p.tokens, warps, rows);
    blocks = gx * rows;
    rc = dispatch(p, dtype, interleaved != 0, true, dim3((unsigned)gx, (unsigned)rows), 32 * warps,
                  stream);
    if (rc != SA_OK) return rc;
  }
  if (!weights) return SA_OK;
  return sa::nr::sum_partial_rows(part, blocks, Hk > 0 ? 2 * D : D, 2 * D, dw_q, dw_k, D, stream);
}
