// qk_norm_rope_bwd.cu — gradient of the hidden-wide Q/K norm + rotation
// (qk_norm_rope.cu), and the sum of partial rows that both norm gradients use.
//
// With g = the rotation transposed applied to the upstream gradient, u = g w
// and r = 1 / sqrt(mean x^2 + eps) over the hidden channels of a row:
//   dx = r (u - x r^2 mean(u x)),   dw = sum over rows of g x r.
// Memory-bound: x and the upstream gradient are read and dx written once
// (6 bf16 values per hidden channel of Q and K together). A block takes whole
// rows, one 8-channel vector of Q and one of K per thread, so that the angles
// are read once for both and dw needs 16 registers. The rows and their angles
// come through a ring of bulk copies, three rows ahead. (A warp per row with 48
// channels a lane needed 158 registers and reached 28% of the copy rate; rows
// loaded one ahead into registers spilled and reached 55%.)

#include <math.h>

#include "norm_rope.cuh"

namespace sa {
namespace nr {

// 32 columns per block, 32 interleaved chains of rows: short enough that the
// loads of a chain are all in flight (8 chains took 10 us for 600 rows).
constexpr int kChains = 32;
__global__ void __launch_bounds__(32 * kChains)
    partial_rows_kernel(const float* part, int rows, int cols, int pitch, float* out0, float* out1,
                        int cols0) {
  __shared__ float red[kChains][33];
  wait_prior_kernel();
  const int l = threadIdx.x & 31, chain = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + l;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int r = chain; r < rows; r += kChains) s += part[(int64_t)r * pitch + c];
  }
  red[chain][l] = s;
  __syncthreads();
  // warp w sums column w of the block over the chains
  s = red[l][chain];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int cw = blockIdx.x * 32 + chain;
  if (l == 0 && cw < cols) {
    if (cw < cols0) out0[cw] = s; else out1[cw - cols0] = s;
  }
}

int sum_partial_rows(const float* part, int rows, int cols, int pitch, float* out0, float* out1,
                     int cols0, cudaStream_t stream) {
  SA_CUDA_TRY(launch_after(partial_rows_kernel, dim3((cols + 31) / 32), dim3(32 * kChains), 0,
                           stream, part, rows, cols, pitch, out0, out1, cols0));
  return SA_OK;
}

}  // namespace nr

namespace qkrope_bwd {

using namespace sa::nr;

constexpr int kMaxHidden = 4096;
constexpr int kMaxThreads = kMaxHidden / 8;
constexpr int kRing = 3;  // rows in flight per block

struct Params {
  const __nv_bfloat16* src[4];  // q, k, and the upstream gradients of both
  int64_t ss[4];
  __nv_bfloat16* o[2];
  int64_t os[2];
  const void* w[2];
  int rows, S, hidden, D;
  int w_dtype;
  float eps;
  const float *cos_t, *sin_t;
  int64_t fs;
  float* part;  // [block][2][hidden], NULL without dw
  int32_t* status;
};

// Four sums over a warp at once: after two exchange steps a lane carries one
// of the four (by its lowest two bits), then they are reduced over the rest.
// Lane l < 4 ends with value l. 6 shuffles where 20 would do one by one.
__device__ __forceinline__ float warp_sum4(float a, float b, float c, float d, int lane) {
  const bool hi = lane & 1, hi2 = lane & 2;
  float x = hi ? b : a, y = hi ? d : c;  // kept: values 0/1 and 2/3 by the lowest bit
  x += __shfl_xor_sync(0xffffffffu, hi ? a : b, 1);
  y += __shfl_xor_sync(0xffffffffu, hi ? c : d, 1);
  float z = hi2 ? y : x;
  z += __shfl_xor_sync(0xffffffffu, hi2 ? x : y, 2);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  return z;
}

// One thread per 8 channels; rows blockIdx.x, + gridDim.x, ... Registers are
// capped so that 768 threads fit an SM.
template <int MAXT>
__global__ void __launch_bounds__(MAXT, 768 / MAXT) kernel(const Params p) {
  __shared__ float sums[2][MAXT / 32 * 4];
  __shared__ __align__(8) uint64_t full[kRing];
  // [kRing] slots: four rows of bf16, then the position's cosines and sines
  extern __shared__ __align__(16) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int c0 = threadIdx.x * 8;
  const bool on = c0 < p.hidden;
  const uint32_t row_bytes = p.hidden * 2, angle_bytes = p.cos_t != nullptr ? p.D * 2 : 0;
  const uint32_t slot_bytes = 4 * row_bytes + 2 * angle_bytes;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  release_next_kernel();
  __syncthreads();
  wait_prior_kernel();
  auto fetch = [&](int slot, int row) {
    uint8_t* dst = ring + slot * slot_bytes;
    mbar_arrive_expect_tx(&full[slot], slot_bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      bulk_load(dst + i * row_bytes, p.src[i] + (int64_t)row * p.ss[i], row_bytes, &full[slot]);
    if (p.cos_t != nullptr) {
      const int64_t at = (int64_t)((unsigned)row % (unsigned)p.S) * p.fs;
      bulk_load(dst + 4 * row_bytes, p.cos_t + at, angle_bytes, &full[slot]);
      bulk_load(dst + 4 * row_bytes + angle_bytes, p.sin_t + at, angle_bytes, &full[slot]);
    }
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < kRing; ++i)
      if ((int64_t)blockIdx.x + (int64_t)i * gridDim.x < p.rows)
        fetch(i, blockIdx.x + i * gridDim.x);
  const int p0 = (c0 % p.D) >> 1;
  const float inv_n = 1.f / (float)p.hidden;
  V8 acc[2] = {fill8(0.f), fill8(0.f)};
  V8 w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = load_weight8(p.w[i], p.w_dtype, on ? c0 : 0);
  int n = 0;  // rows done
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, ++n) {
    const int slot = n % kRing;
    const uint8_t* src = ring + slot * slot_bytes;
    // the rows arrive by themselves: a copy that does not leaves NaN behind
    const bool there = mbar_wait(&full[slot], (uint32_t)(n / kRing) & 1u, p.status, nullptr);
    float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.cos_t != nullptr && on) {
      const uint8_t* angles = src + 4 * row_bytes + p0 * 4;
      c4 = *reinterpret_cast<const float4*>(angles);
      s4 = *reinterpret_cast<const float4*>(angles + angle_bytes);
    }
    const uint64_t c2[2] = {f2_pack(c4.x, c4.y), f2_pack(c4.z, c4.w)};
    const uint64_t s2[2] = {f2_pack(s4.x, s4.y), f2_pack(s4.z, s4.w)};
    const uint64_t n2[2] = {f2_pack(-s4.x, -s4.y), f2_pack(-s4.z, -s4.w)};
    V8 x[2], g[2];
    float ss[2], dot[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      Raw8<__nv_bfloat16> rx = {}, rd = {};
      if (on) {
        rx.v[0] = reinterpret_cast<const uint4*>(src + i * row_bytes)[threadIdx.x];
        rd.v[0] = reinterpret_cast<const uint4*>(src + (2 + i) * row_bytes)[threadIdx.x];
      }
      x[i] = unpack8(rx);
      const V8 d = unpack8(rd);
      uint64_t a2 = 0ull, b2 = 0ull;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        g[i].v[2 * j] = f2_fma(d.v[2 * j], c2[j], f2_mul(d.v[2 * j + 1], s2[j]));
        g[i].v[2 * j + 1] = f2_fma(d.v[2 * j + 1], c2[j], f2_mul(d.v[2 * j], n2[j]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a2 = f2_fma(x[i].v[j], x[i].v[j], a2);
        b2 = f2_fma(f2_mul(g[i].v[j], w[i].v[j]), x[i].v[j], b2);
      }
      ss[i] = sum2(a2);
      dot[i] = sum2(b2);
    }
    const float z = warp_sum4(ss[0], dot[0], ss[1], dot[1], lane);
    // two buffers in turn: a warp writes a row's sums only after the block has
    // passed the barrier of the row before, so the row before that has been read
    float* turn = sums[n & 1];
    if (lane < 4) turn[warp * 4 + lane] = z;
    __syncthreads();
    // every thread has its part of the row in registers: the slot is free
    if (threadIdx.x == 0 && row + (int64_t)kRing * gridDim.x < p.rows) {
      fence_proxy_async_smem();
      fetch(slot, (int)(row + (int64_t)kRing * gridDim.x));
    }
    // lane l sums value l & 3 of every eighth warp, then over the lanes
    float t = 0.f;
    for (int v = lane; v < warps * 4; v += 32) t += turn[v];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float sq = __shfl_sync(0xffffffffu, t, 2 * i);
      const float dt = __shfl_sync(0xffffffffu, t, 2 * i + 1);
      float r = inv_sqrt<__nv_bfloat16>(fmaf(sq, inv_n, p.eps));
      if (!there) r = __int_as_float(0x7fc00000);
      // the dot product first: r^3 alone leaves fp32 where x is about 1e14 or 1e-13
      const float m = -(r * dt * inv_n) * r * r;
      const uint64_t r2 = f2_pack(r, r), m2 = f2_pack(m, m);
      V8 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t gr = f2_mul(g[i].v[j], r2);
        acc[i].v[j] = f2_fma(gr, x[i].v[j], acc[i].v[j]);
        o.v[j] = f2_fma(x[i].v[j], m2, f2_mul(gr, w[i].v[j]));
      }
      if (on) store8(p.o[i] + row * p.os[i] + c0, o);
    }
  }
  if (p.part == nullptr || !on) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    store8(p.part + ((int64_t)blockIdx.x * 2 + i) * p.hidden + c0, acc[i]);
}

// Blocks: 768 threads per SM, and at least two rows each where there
// are that few, as every block leaves a partial row of dw to be read again.
int blocks_of(int rows, int threads) {
  const int per_sm = 768 / threads > 1 ? 768 / threads : 1;
  const int64_t most = (int64_t)sa::sm_count_current_device() * (per_sm < 16 ? per_sm : 16);
  const int64_t want = ((int64_t)rows + 1) / 2;
  return (int)(want < most ? want : most);
}

int threads_of(int hidden) { return (hidden / 8 + 31) / 32 * 32; }

}  // namespace qkrope_bwd
}  // namespace sa

extern "C" size_t sa_qk_norm_rope_bwd_workspace_size(int hidden) {
  if (hidden < 8 || hidden > sa::qkrope_bwd::kMaxHidden) return 0;
  using namespace sa::qkrope_bwd;
  return (size_t)blocks_of(0x7ffffffe, threads_of(hidden)) * 2 * hidden * sizeof(float);
}

extern "C" int sa_qk_norm_rope_bwd(const void* dq, const void* dk, int64_t dq_row_stride,
                                   int64_t dk_row_stride, const void* q, const void* k,
                                   int64_t q_row_stride, int64_t k_row_stride, int rows, int S,
                                   int hidden, int D, const void* w_q, const void* w_k,
                                   int w_is_bf16, float eps, const float* cos_table,
                                   const float* sin_table, int64_t freq_row_stride, void* dq_in,
                                   void* dk_in, int64_t dqi_row_stride, int64_t dki_row_stride,
                                   float* dw_q, float* dw_k, void* workspace, size_t ws_bytes,
                                   int32_t* status, cudaStream_t stream) {
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
    p.src[0] = static_cast<const __nv_bfloat16*>(q); p.ss[0] = q_row_stride;
    p.src[1] = static_cast<const __nv_bfloat16*>(k); p.ss[1] = k_row_stride;
    p.src[2] = static_cast<const __nv_bfloat16*>(dq); p.ss[2] = dq_row_stride;
    p.src[3] = static_cast<const __nv_bfloat16*>(dk); p.ss[3] = dk_row_stride;
    p.o[0] = static_cast<__nv_bfloat16*>(dq_in); p.os[0] = dqi_row_stride;
    p.o[1] = static_cast<__nv_bfloat16*>(dk_in); p.os[1] = dki_row_stride;
    p.w[0] = w_q; p.w[1] = w_k;
    p.rows = rows; p.S = S; p.hidden = hidden; p.D = D;
    p.w_dtype = w_is_bf16 ? SA_DTYPE_BF16 : SA_DTYPE_FP32;
    p.eps = eps;
    p.cos_t = cos_table; p.sin_t = sin_table; p.fs = freq_row_stride;
    p.part = dw_q != nullptr ? part : nullptr;
    const int threads = threads_of(hidden);
    part_rows = blocks_of(rows, threads);
    p.status = status;
    const size_t smem = (size_t)kRing * (4 * hidden * 2 + (cos_table != nullptr ? 4 * D : 0));
    const void* fn_ptr = threads <= 256 ? (const void*)kernel<256> : (const void*)kernel<kMaxThreads>;
    const int rc = sa::func_attr_once(fn_ptr, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      // rows and angles of the widest head, D = hidden
                                      kRing * (4 * 2 + 4) * 8 * (threads <= 256 ? 256 : kMaxThreads));
    if (rc != SA_OK) return rc;
    SA_CUDA_TRY(sa::launch_after(threads <= 256 ? kernel<256> : kernel<kMaxThreads>,
                                 dim3(part_rows), dim3(threads), smem, stream, p));
  }
  if (dw_q == nullptr) return SA_OK;
  return sa::nr::sum_partial_rows(part, part_rows, 2 * hidden, 2 * hidden, dw_q, dw_k, hidden,
                                  stream);
}
