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
// the sums are shuffles inside a lane group. A warp walks heads of one token
// and one tensor, loading a few heads ahead, and folds weight, cosine and sine
// into the two factors of each channel once for all of them; the arithmetic is
// f32x2. Everything between the load and the store is fp32: the one rounding is
// that of the result.

#include <math.h>

#include "norm_rope.cuh"

namespace sa {
namespace headnorm {

using namespace sa::nr;

// Heads of a lane group in flight, about 64 KB per SM with the warps that fit.
template <typename T>
__host__ __device__ constexpr int ahead() { return sizeof(T) == 2 ? 3 : 2; }
constexpr int kAheadBwd = 4;
constexpr int kWarps = 8;        // of a block
constexpr int kMaxHeads = 8192;  // of q and k together

// [0] q, [1] k. Head strides are 32-bit: a head's offset is one multiply-add.
struct Tensors {
  const void* base[2];
  int64_t s0[2], s1[2];  // batch, sequence
  int s2[2];             // head
};

struct Params {
  Tensors x, o, d;  // inputs, outputs, upstream gradients (gradient only)
  int B, S, Hq, Hk, D, rot;
  const void* w[2];
  int w_dtype;
  float eps;
  const float *cos_t, *sin_t;
  int64_t fs;
  int table_rows;
  const void* pos;
  int pos_i64;
  int64_t ps0, ps1;
  int steps;             // of a warp, 32 / G heads each
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

template <typename T>
__device__ __forceinline__ const T* token_ptr(const Tensors& t, int which, const Token& k) {
  return reinterpret_cast<const T*>(t.base[which]) + k.b * t.s0[which] + k.s * t.s1[which];
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
      c4 = *reinterpret_cast<const float4*>(p.cos_t + row * p.fs + (c0 >> 1));
      s4 = *reinterpret_cast<const float4*>(p.sin_t + row * p.fs + (c0 >> 1));
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
        const float4 c4 = *reinterpret_cast<const float4*>(p.cos_t + row * p.fs + i0 + i);
        const float4 s4 = *reinterpret_cast<const float4*>(p.sin_t + row * p.fs + i0 + i);
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

// This warp's heads: tensor (0 q, 1 k), those of its lane group (first, end,
// 32 / G apart).
struct Heads {
  int which, first, end;
};

template <int G>
__device__ __forceinline__ Heads heads_of(const Params& p, int chunk, int lane) {
  Heads h;
  h.which = chunk >= p.chunks_q ? 1 : 0;
  const int c = h.which ? chunk - p.chunks_q : chunk, per = p.steps * (32 / G);
  h.first = c * per + lane / G;
  h.end = min(h.which ? p.Hk : p.Hq, (c + 1) * per);
  return h;
}

// One warp per token and chunk of heads.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kWarps, INTER ? 4 : 3) fwd_kernel(const Params p) {
  constexpr int kAhead = ahead<T>();
  const int lane = threadIdx.x & 31;
  const unsigned gw = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const unsigned t = gw / (unsigned)p.chunks;
  release_next_kernel();  // calls in a row overlap start and end (fp32, 2 x 1333: 10.2 -> 8.3 us)
  wait_prior_kernel();
  if (t >= (unsigned)p.tokens) return;
  const Heads hd = heads_of<G>(p, gw - t * p.chunks, lane);
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  const Token tk = token_of(p, t);
  const T* src = token_ptr<T>(p.x, hd.which, tk) + c0;
  T* dst = const_cast<T*>(token_ptr<T>(p.o, hd.which, tk)) + c0;
  const int hs = p.x.s2[hd.which], ohs = p.o.s2[hd.which];
  auto load = [&](int h) {
    Raw8<T> r = {};
    if (on && h < hd.end) r = load8(src + (int64_t)h * hs);
    return r;
  };
  Raw8<T> raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) raw[i] = load(hd.first + i * (32 / G));
  int pc0;
  const int partner = partner_of<INTER>(p, lane, c0, pc0);
  const void* wp = p.w[hd.which];
  const V8 w = load_weight8(wp, p.w_dtype, on ? c0 : 0);
  const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, 1.f);
  // out = r (x a + other b) per channel, other = the pair's second channel
  V8 a, b;
  if (INTER) {
    const uint64_t minus = f2_pack(-1.f, -1.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
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
  // lane groups whose heads run out keep step with the warp
  for (int base = hd.first - lane / G; base < hd.end; base += kAhead * (32 / G)) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int h = base + i * (32 / G) + lane / G;
      const Raw8<T> cur = raw[i];
      raw[i] = load(h + kAhead * (32 / G));
      const V8 x = unpack8(cur);
      uint64_t s2 = f2_mul(x.v[0], x.v[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) s2 = f2_fma(x.v[j], x.v[j], s2);
      const float ss = group_sum<G>(sum2(s2));
      float r = inv_sqrt<T>(fmaf(ss, inv_d, p.eps));
      if (tk.bad) r = __int_as_float(0x7fc00000);
      const uint64_t r2 = f2_pack(r, r);
      V8 other;
      if (INTER) {
        other = V8{{x.v[1], x.v[0], x.v[3], x.v[2]}};
      } else {
        other = unpack8(shfl8(cur, partner));
      }
      V8 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o.v[j] = f2_mul(f2_fma(x.v[j], a.v[j], f2_mul(other.v[j], b.v[j])), r2);
      if (on && h < hd.end) store8(dst + (int64_t)h * ohs, o);
    }
  }
}

// Gradient: a warp keeps its chunk of heads and walks the tokens with a fixed
// stride, so that its part of dw stays in registers; a block writes one partial
// row.
template <typename T, int G, bool INTER>
__global__ void __launch_bounds__(32 * kWarps, 2) bwd_kernel(const Params p) {
  __shared__ float red[kWarps][G * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned gw = blockIdx.x * kWarps + warp;
  const unsigned t0 = gw / (unsigned)p.chunks, step = gridDim.x * kWarps / (unsigned)p.chunks;
  const Heads hd = heads_of<G>(p, gw - t0 * p.chunks, lane);
  const int c0 = (lane % G) * 8;
  const bool on = c0 < p.D;
  int pc0;
  const int partner = partner_of<INTER>(p, lane, c0, pc0);
  wait_prior_kernel();
  const V8 w = load_weight8(p.w[hd.which], p.w_dtype, on ? c0 : 0);
  const int xs2 = p.x.s2[hd.which], ds2 = p.d.s2[hd.which], os2 = p.o.s2[hd.which];
  release_next_kernel();
  V8 acc = fill8(0.f);
  const float inv_d = 1.f / (float)p.D;
  if (t0 < step) {  // warps past the last whole set of chunks have no tokens
    for (unsigned t = t0; t < (unsigned)p.tokens; t += step) {
      const Token tk = token_of(p, t);
      const T* xt = token_ptr<T>(p.x, hd.which, tk) + c0;
      const T* dt = token_ptr<T>(p.d, hd.which, tk) + c0;
      T* ot = const_cast<T*>(token_ptr<T>(p.o, hd.which, tk)) + c0;
      Raw8<T> rx[kAheadBwd], rd[kAheadBwd];
      auto load = [&](int i, int h) {
        rx[i] = rd[i] = Raw8<T>{};
        if (on && h < hd.end) {
          rx[i] = load8(xt + (int64_t)h * xs2);
          rd[i] = load8(dt + (int64_t)h * ds2);
        }
      };
#pragma unroll
      for (int i = 0; i < kAheadBwd; ++i) load(i, hd.first + i * (32 / G));
      const Angles<INTER> ang = load_angles<INTER>(p, tk.row, c0, -1.f);
      const uint64_t minus = f2_pack(-1.f, -1.f);
      const uint64_t pos_s[2] = {f2_mul(ang.s[0], minus), f2_mul(ang.s[1], minus)};
      if (tk.bad && lane == 0) report_status(p.status, SA_DEV_BAD_INDEX);
      for (int base = hd.first - lane / G; base < hd.end; base += kAheadBwd * (32 / G)) {
#pragma unroll
        for (int i = 0; i < kAheadBwd; ++i) {
          const int h = base + i * (32 / G) + lane / G;
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
          load(i, h + kAheadBwd * (32 / G));
          uint64_t s2 = f2_mul(x.v[0], x.v[0]);
          uint64_t t2 = f2_mul(f2_mul(g.v[0], w.v[0]), x.v[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) {
            s2 = f2_fma(x.v[j], x.v[j], s2);
            t2 = f2_fma(f2_mul(g.v[j], w.v[j]), x.v[j], t2);
          }
          const float ss = group_sum<G>(sum2(s2)), dot = group_sum<G>(sum2(t2));
          float r = inv_sqrt<T>(fmaf(ss, inv_d, p.eps));
          if (tk.bad) r = __int_as_float(0x7fc00000);
          // the dot product first: r^3 alone leaves fp32 where x is about 1e14 or 1e-13
          const float m = -(r * dot * inv_d) * r * r;
          const uint64_t r2 = f2_pack(r, r), m2 = f2_pack(m, m);
          if (on && h < hd.end) {
            V8 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint64_t gr = f2_mul(g.v[j], r2);
              acc.v[j] = f2_fma(gr, x.v[j], acc.v[j]);
              o.v[j] = f2_fma(x.v[j], m2, f2_mul(gr, w.v[j]));
            }
            store8(ot + (int64_t)h * os2, o);
          }
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
  __shared__ int tensor[kWarps];
  if (lane == 0) tensor[warp] = hd.which;
  __syncthreads();
  float* row = p.part + (int64_t)blockIdx.x * 2 * p.D;
  for (int c = threadIdx.x; c < 2 * p.D; c += 32 * kWarps) {
    const int which = c >= p.D, cc = which ? c - p.D : c;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v)
      if (tensor[v] == which) s += red[v][cc];
    row[c] = s;
  }
}

template <typename T, int G>
cudaError_t launch_g(const Params& p, bool inter, bool bwd, int grid, cudaStream_t stream) {
  const auto kernel = bwd ? inter ? bwd_kernel<T, G, true> : bwd_kernel<T, G, false>
                          : inter ? fwd_kernel<T, G, true> : fwd_kernel<T, G, false>;
  return launch_after(kernel, dim3(grid), dim3(32 * kWarps), 0, stream, p);
}

// lanes of a head: the power of two that covers D / 8, at least 4
int group_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

template <typename T>
cudaError_t launch_t(const Params& p, bool inter, bool bwd, int grid, cudaStream_t stream) {
  switch (group_of(p.D)) {
    case 4: return launch_g<T, 4>(p, inter, bwd, grid, stream);
    case 8: return launch_g<T, 8>(p, inter, bwd, grid, stream);
    case 16: return launch_g<T, 16>(p, inter, bwd, grid, stream);
    default: return launch_g<T, 32>(p, inter, bwd, grid, stream);
  }
}

int dispatch(const Params& p, int dtype, bool inter, bool bwd, int grid, cudaStream_t stream) {
  if (dtype == SA_DTYPE_BF16) SA_CUDA_TRY(launch_t<__nv_bfloat16>(p, inter, bwd, grid, stream));
  else if (dtype == SA_DTYPE_FP16) SA_CUDA_TRY(launch_t<__half>(p, inter, bwd, grid, stream));
  else SA_CUDA_TRY(launch_t<float>(p, inter, bwd, grid, stream));
  return SA_OK;
}

// Chunks of heads: as long as leaves `want` warps over all tokens (the angles
// and factors of a token are then worked out by fewer warps), at least `ahead`
// steps.
void shape(Params& p, int ahead, int64_t want) {
  const int per = 32 / group_of(p.D);
  const int sq = (p.Hq + per - 1) / per, sk = (p.Hk + per - 1) / per;
  const auto chunks = [&](int steps) {
    return (sq + steps - 1) / steps + (sk + steps - 1) / steps;
  };
  p.steps = ahead;
  while (p.steps < (sq > sk ? sq : sk) && p.tokens * (int64_t)chunks(2 * p.steps) >= want)
    p.steps *= 2;
  p.chunks_q = (sq + p.steps - 1) / p.steps;
  p.chunks = chunks(p.steps);
}

// The gradient's blocks, each a partial row of dw: 16 warps per SM, in whole
// sets of chunks (the last few warps may have no tokens).
constexpr int kBwdBlocksPerSm = 2;
int bwd_grid(const Params& p) {
  const int64_t want = ((int64_t)p.tokens * p.chunks + kWarps - 1) / kWarps;
  const int64_t least = (p.chunks + kWarps - 1) / kWarps;  // a warp for every chunk
  int64_t most = (int64_t)sa::sm_count_current_device() * kBwdBlocksPerSm;
  if (most < least) most = least;
  return (int)(want < most ? want : most);
}

bool aligned_ok(const void* base, const int64_t st[4], int dtype) {
  if (base == nullptr) return true;
  const int64_t mult = dtype == SA_DTYPE_FP32 ? 4 : 8;
  return (uintptr_t)base % 16 == 0 && st != nullptr && st[3] == 1 && st[0] >= 0 && st[1] >= 0 &&
         st[2] >= 0 && st[0] % mult == 0 && st[1] % mult == 0 && st[2] % mult == 0 &&
         st[2] <= 0x7fffffff;
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

Tensors tensors(const void* q, const void* k, const int64_t* qs, const int64_t* ks) {
  return Tensors{{q, k}, {qs[0], ks[0]}, {qs[1], ks[1]}, {(int)qs[2], (int)ks[2]}};
}

void common(Params& p, const void* q, const void* k, const int64_t* qs, const int64_t* ks, int B,
            int S, int Hq, int Hk, int D, const void* w_q, const void* w_k, int w_dtype, float eps,
            const float* cos_t, const float* sin_t, int64_t fs, int table_rows, int rot,
            const void* positions, int pos_i64, const int64_t* pos_strides, void* qo, void* ko,
            const int64_t* qos, const int64_t* kos, int32_t* status) {
  static const int64_t zero[4] = {0, 0, 0, 1};
  if (Hk == 0) ks = kos = zero;
  p = Params{};
  p.x = tensors(q, k, qs, ks);
  p.o = tensors(qo, ko, qos, kos);
  p.B = B; p.S = S; p.Hq = Hq; p.Hk = Hk; p.D = D;
  p.rot = cos_t != nullptr ? rot : 0;
  p.w[0] = w_q; p.w[1] = w_k; p.w_dtype = w_dtype; p.eps = eps;
  p.cos_t = cos_t; p.sin_t = sin_t; p.fs = fs; p.table_rows = table_rows;
  p.pos = positions; p.pos_i64 = pos_i64;
  if (positions != nullptr) { p.ps0 = pos_strides[0]; p.ps1 = pos_strides[1]; }
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
         q_out, k_out, qo_strides, ko_strides, status);
  shape(p, dtype == SA_DTYPE_FP32 ? ahead<float>() : ahead<__half>(),
        (int64_t)sa::sm_count_current_device() * 64);
  const int64_t blocks = ((int64_t)p.tokens * p.chunks + kWarps - 1) / kWarps;
  SA_CHECK_ARG(blocks <= 0x7fffffff / kWarps, "%s: too many tokens", fn);
  return dispatch(p, dtype, interleaved != 0, false, (int)blocks, stream);
}

extern "C" size_t sa_qk_head_norm_rope_bwd_workspace_size(int D) {
  if (D < 8) return 0;
  const int64_t most = (int64_t)sa::sm_count_current_device() * sa::headnorm::kBwdBlocksPerSm;
  const int64_t least =
      sa::headnorm::kMaxHeads / (sa::headnorm::kAheadBwd * sa::headnorm::kWarps) + 1;
  return (size_t)(most > least ? most : least) * 2 * D * sizeof(float);
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
    p.d = tensors(dq, dk, dq_strides, Hk > 0 ? dk_strides : dq_strides);
    p.part = weights ? part : nullptr;
    shape(p, kAheadBwd, (int64_t)sa::sm_count_current_device() * kBwdBlocksPerSm * kWarps * 2);
    SA_CHECK_ARG((int64_t)p.tokens * p.chunks <= 0x7fffffff, "%s: too many tokens", fn);
    blocks = bwd_grid(p);
    rc = dispatch(p, dtype, interleaved != 0, true, blocks, stream);
    if (rc != SA_OK) return rc;
  }
  if (!weights) return SA_OK;
  return sa::nr::sum_partial_rows(part, blocks, Hk > 0 ? 2 * D : D, 2 * D, dw_q, dw_k, D, stream);
}
