// LayerNorm over the last axis, forward and backward, fp16 / bf16 / fp32 rows of any length.
//
//   forward   m = sum(x) / C,  r = 1 / sqrt(sum((x - m)^2) / C + eps),  y = (x - m) r w + b
//   backward  h = (x - m) r,  g = dy w:  dx = r (g - mean(g) - h mean(g h)),
//             dw = sum over rows of dy h,  db = sum over rows of dy
//
// Bound by memory: the forward pass reads x and writes y once, the backward pass reads dy and x and writes dx once.  A row
// therefore stays in registers (as loaded, not widened) between its reduction and its result: one warp holds a short
// row, a block a long one, and only rows longer than a block's registers are read again.  Sums are fp32; the variance is
// taken of the differences from the mean.  dw and db: every thread keeps the sums of its own columns over all rows that it
// meets, a block adds those of its warps, and a second launch adds the blocks' in a fixed order (no atomics).
#include "bxl_common.cuh"
#include "bxl_host.h"
#include "bxl_types.cuh"

namespace bxl {

struct LnArgs {
  const void *x, *dy;
  void* y;                  // forward: result; backward: dx
  long long ldx, lddy, ldy;
  const void *weight, *bias;
  float *mean, *rstd;       // forward: written (or null); backward: read
  float* part;              // backward: [blocks][2][C] column sums of dy h and of dy, or null
  long long rows;
  int C, param_f32;
  float eps, inv_c;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block; every thread gets it.  `slot` has one float per warp; two reductions in a row take different slots,
// so that one barrier each is enough.
__device__ __forceinline__ float block_sum(float v, float* slot) {
  v = warp_sum(v);
  const int lane = threadIdx.x & 31;
  if (lane == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < static_cast<int>(blockDim.x >> 5) ? slot[lane] : 0.f);
}

constexpr int kLnWarps = 8;   // rows in flight in a block of the warp-per-row form

// kWarp: a warp per row, kLnWarps rows per block.  Otherwise a block per row.  NV vectors of VEC elements per thread.
template <class T, int VEC, int NV, bool kWarp>
__global__ void __launch_bounds__(kWarp ? kLnWarps * 32 : 1024) ln_fwd_kernel(const LnArgs a) {
  pdl_launch_dependents();
  __shared__ float red[2][32];
  const int tid = kWarp ? (threadIdx.x & 31) : threadIdx.x;
  const int step = kWarp ? 32 : blockDim.x;
  const int n = a.C / VEC;
  const Param<T> w{a.weight, a.param_f32}, b{a.bias, a.param_f32};
  const long long first = kWarp ? blockIdx.x * (long long)kLnWarps + (threadIdx.x >> 5) : blockIdx.x;
  const long long stride = kWarp ? gridDim.x * (long long)kLnWarps : gridDim.x;
  pdl_wait();
  for (long long r = first; r < a.rows; r += stride) {
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    Vec<T, VEC> raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) raw[i] = load_vec<T, VEC>(xr + (tid + i * step) * VEC);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += to_f32(raw[i].v[j]);
      }
    const float mean = (kWarp ? warp_sum(s) : block_sum(s, red[0])) / a.C;   // a division: the mean of equal values is their value
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = to_f32(raw[i].v[j]) - mean;
          q = fmaf(d, d, q);
        }
      }
    const float rstd = rsqrtf((kWarp ? warp_sum(q) : block_sum(q, red[1])) * a.inv_c + a.eps);
    T* yr = static_cast<T*>(a.y) + r * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (tid + i * step) * VEC;
      if (tid + i * step < n) {
        float wv[VEC], bv[VEC];
        if (w.p) w.template get<VEC>(c, wv);
        if (b.p) b.template get<VEC>(c, bv);
        Vec<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float h = (to_f32(raw[i].v[j]) - mean) * rstd;
          o.v[j] = from_f32<T>(fmaf(h, w.p ? wv[j] : 1.f, b.p ? bv[j] : 0.f));
        }
        store_vec<T, VEC>(yr + c, o);
      }
    }
    if (a.mean && tid == 0) a.mean[r] = mean, a.rstd[r] = rstd;
  }
}

// Rows longer than a block's registers: three passes over the row, the second and third mostly from L2.
template <class T>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const LnArgs a) {
  pdl_launch_dependents();
  __shared__ float red[2][32];
  const Param<T> w{a.weight, a.param_f32}, b{a.bias, a.param_f32};
  pdl_wait();
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) s += to_f32(xr[c]);
    const float mean = block_sum(s, red[0]) / a.C;
    float q = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float d = to_f32(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = rsqrtf(block_sum(q, red[1]) * a.inv_c + a.eps);
    T* yr = static_cast<T*>(a.y) + r * a.ldy;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x)
      yr[c] = from_f32<T>(fmaf((to_f32(xr[c]) - mean) * rstd, w.p ? w.at(c) : 1.f, b.p ? b.at(c) : 0.f));
    if (a.mean && threadIdx.x == 0) a.mean[r] = mean, a.rstd[r] = rstd;
  }
}

// ---- backward ------------------------------------------------------------------------------
// The next row of dy and x is on its way while the present one is reduced.
template <class T, int VEC, int NV, bool kWarp>
__global__ void __launch_bounds__(kWarp ? kLnWarps * 32 : (NV * VEC > 8 ? 512 : 1024)) ln_bwd_kernel(const LnArgs a) {
  pdl_launch_dependents();
  extern __shared__ float4 dyn[];                       // weight [C]; afterwards the warps' column sums
  float* sw = reinterpret_cast<float*>(dyn);
  __shared__ float red[2][2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = kWarp ? lane : threadIdx.x;
  const int step = kWarp ? 32 : blockDim.x;
  const int n = a.C / VEC;
  const Param<T> w{a.weight, a.param_f32};
  pdl_wait();
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) sw[c] = w.p ? w.at(c) : 1.f;
  __syncthreads();
  const long long first = kWarp ? blockIdx.x * (long long)kLnWarps + warp : blockIdx.x;
  const long long stride = kWarp ? gridDim.x * (long long)kLnWarps : gridDim.x;
  float dw[NV * VEC], db[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) dw[i] = db[i] = 0.f;
  Vec<T, VEC> x[NV], dy[NV], xn[NV], dyn_[NV];
  float mean = 0.f, rstd = 0.f, mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](long long r, Vec<T, VEC>(&xv)[NV], Vec<T, VEC>(&dv)[NV], float& m, float& s) {
    if (r >= a.rows) return;
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dr = static_cast<const T*>(a.dy) + r * a.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
        xv[i] = load_vec<T, VEC>(xr + (tid + i * step) * VEC);
        dv[i] = load_vec<T, VEC>(dr + (tid + i * step) * VEC);
      }
    m = a.mean[r], s = a.rstd[r];
  };
  fetch(first, x, dy, mean, rstd);
  int it = 0;
  for (long long r = first; r < a.rows; r += stride, it ^= 1) {
    fetch(r + stride, xn, dyn_, mean_n, rstd_n);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = to_f32(dy[i].v[j]), h = (to_f32(x[i].v[j]) - mean) * rstd;
          const float g = d * sw[(tid + i * step) * VEC + j];
          s1 += g;
          s2 = fmaf(g, h, s2);
          db[i * VEC + j] += d;
          dw[i * VEC + j] = fmaf(d, h, dw[i * VEC + j]);
        }
      }
    s1 = warp_sum(s1), s2 = warp_sum(s2);
    if (!kWarp) {
      if (lane == 0) red[it][0][warp] = s1, red[it][1][warp] = s2;
      __syncthreads();
      const bool in = lane < static_cast<int>(blockDim.x >> 5);
      s1 = warp_sum(in ? red[it][0][lane] : 0.f), s2 = warp_sum(in ? red[it][1][lane] : 0.f);
    }
    s1 *= a.inv_c, s2 *= a.inv_c;
    T* out = static_cast<T*>(a.y) + r * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
        Vec<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float h = (to_f32(x[i].v[j]) - mean) * rstd;
          const float g = to_f32(dy[i].v[j]) * sw[(tid + i * step) * VEC + j];
          o.v[j] = from_f32<T>(rstd * (g - s1 - h * s2));
        }
        store_vec<T, VEC>(out + (tid + i * step) * VEC, o);
      }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = xn[i], dy[i] = dyn_[i];
    mean = mean_n, rstd = rstd_n;
  }
  if (!a.part) return;
  float* pw = a.part + blockIdx.x * 2ll * a.C;
  if (kWarp) {
    // the warps' sums, added pairwise through shared memory
    for (int half = kLnWarps / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (warp >= half && warp < 2 * half) {
        float* to = sw + (warp - half) * 2ll * a.C;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (tid + i * step < n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) to[(tid + i * step) * VEC + j] = dw[i * VEC + j], to[a.C + (tid + i * step) * VEC + j] = db[i * VEC + j];
          }
      }
      __syncthreads();
      if (warp < half) {
        const float* from = sw + warp * 2ll * a.C;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (tid + i * step < n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) dw[i * VEC + j] += from[(tid + i * step) * VEC + j], db[i * VEC + j] += from[a.C + (tid + i * step) * VEC + j];
          }
      }
    }
    if (warp != 0) return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (tid + i * step < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) pw[(tid + i * step) * VEC + j] = dw[i * VEC + j], pw[a.C + (tid + i * step) * VEC + j] = db[i * VEC + j];
    }
}

// Rows longer than a block's registers: dx alone, two passes over the row.
template <class T>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(const LnArgs a) {
  pdl_launch_dependents();
  __shared__ float red[2][32];
  const Param<T> w{a.weight, a.param_f32};
  pdl_wait();
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dr = static_cast<const T*>(a.dy) + r * a.lddy;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float g = to_f32(dr[c]) * (w.p ? w.at(c) : 1.f);
      s1 += g;
      s2 = fmaf(g, (to_f32(xr[c]) - mean) * rstd, s2);
    }
    s1 = block_sum(s1, red[0]) * a.inv_c;
    s2 = block_sum(s2, red[1]) * a.inv_c;
    T* out = static_cast<T*>(a.y) + r * a.ldy;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float g = to_f32(dr[c]) * (w.p ? w.at(c) : 1.f);
      out[c] = from_f32<T>(rstd * (g - s1 - (to_f32(xr[c]) - mean) * rstd * s2));
    }
  }
}
// ... and their column sums: a thread per column, gridDim.y shares of the rows.
template <class T>
__global__ void __launch_bounds__(256) ln_bwd_columns_kernel(const LnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.f, db = 0.f;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float d = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
    dw = fmaf(d, (to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r], dw);
    db += d;
  }
  a.part[blockIdx.y * 2ll * a.C + c] = dw, a.part[(blockIdx.y * 2ll + 1) * a.C + c] = db;
}

// Adds column sums that blocks have left: 32 columns of one of the two results per block, a warp per share of the partials.
template <class P>
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* part, int count, long long pitch, int C, P* out0, P* out1) {
  pdl_launch_dependents();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  P* out = blockIdx.y ? out1 : out0;
  pdl_wait();
  if (!out) return;
  float v = 0.f;
  if (c < C)
    for (int i = warp; i < count; i += warps) v += part[i * pitch + blockIdx.y * (long long)C + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp) return;
  for (int i = 1; i < warps; ++i) v += s[i][lane];
  if (c < C) out[c] = from_f32<P>(v);
}

int sum_partials(const float* part, int count, long long pitch, int C, void* out0, void* out1, int dtype, cudaStream_t s) {
  const dim3 grid((C + 31) / 32, out1 ? 2 : 1), block(count >= 32 ? 1024 : 128);
  if (dtype == BXL_F32)
    return launch_kernel("sum_partials_kernel launch", sum_partials_kernel<float>, grid, block, 0, s, 1, part, count, pitch, C, static_cast<float*>(out0), static_cast<float*>(out1));
  if (dtype == BXL_F16)
    return launch_kernel("sum_partials_kernel launch", sum_partials_kernel<__half>, grid, block, 0, s, 1, part, count, pitch, C, static_cast<__half*>(out0), static_cast<__half*>(out1));
  return launch_kernel("sum_partials_kernel launch", sum_partials_kernel<__nv_bfloat16>, grid, block, 0, s, 1, part, count, pitch, C,
                       static_cast<__nv_bfloat16*>(out0), static_cast<__nv_bfloat16*>(out1));
}

// ---- host side -----------------------------------------------------------------------------
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kLnMaxC = 1 << 30;   // column indices, and a step past the last one, are ints
constexpr int kLnBlocksPerSm = 4;
// Blocks of the backward pass, each of which leaves one row of column sums: at most four an SM, and no more than one for
// sixteen rows unless that leaves SMs idle (the sums are 16 bytes a column and block, written and read again).
static long long ln_bwd_blocks(long long rows) {
  const long long sms = sm_count();
  long long g = rows / 16 > sms ? rows / 16 : sms;
  if (g > sms * kLnBlocksPerSm) g = sms * kLnBlocksPerSm;
  return g < rows ? g : rows;
}

template <class T, int VEC, int NV, bool kWarp>
static int ln_fwd_launch(const LnArgs& a, int threads, cudaStream_t s) {
  const long long need = kWarp ? (a.rows + kLnWarps - 1) / kLnWarps : a.rows, most = (long long)sm_count() * 16;
  return launch_kernel("ln_fwd_kernel launch", ln_fwd_kernel<T, VEC, NV, kWarp>, dim3((unsigned)(need < most ? need : most)), dim3(threads), 0, s, 1, a);
}
template <class T>
static int ln_fwd(const LnArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    const int n = a.C / V;
    if (n <= 32) return ln_fwd_launch<T, V, 1, true>(a, kLnWarps * 32, s);
    if (n <= 64) return ln_fwd_launch<T, V, 2, true>(a, kLnWarps * 32, s);
    if (n <= 96) return ln_fwd_launch<T, V, 3, true>(a, kLnWarps * 32, s);
    if (n <= 160) return ln_fwd_launch<T, V, 5, true>(a, kLnWarps * 32, s);
    if (n <= 512) return ln_fwd_launch<T, V, 2, false>(a, 256, s);
    if (n <= 1024) return ln_fwd_launch<T, V, 2, false>(a, 512, s);
    if (n <= 2048) return ln_fwd_launch<T, V, 4, false>(a, 512, s);
    if (n <= 8192) return ln_fwd_launch<T, V, 8, false>(a, 1024, s);
  } else {
    if (a.C <= 64) return ln_fwd_launch<T, 1, 2, true>(a, kLnWarps * 32, s);
    if (a.C <= 256) return ln_fwd_launch<T, 1, 8, true>(a, kLnWarps * 32, s);
    if (a.C <= 2048) return ln_fwd_launch<T, 1, 8, false>(a, 256, s);
    if (a.C <= 8192) return ln_fwd_launch<T, 1, 8, false>(a, 1024, s);
    if (a.C <= 16384) return ln_fwd_launch<T, 1, 16, false>(a, 1024, s);
  }
  const long long most = (long long)sm_count() * 2;
  return launch_kernel("ln_fwd_long_kernel launch", ln_fwd_long_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(1024), 0, s, 1, a);
}

template <class T, int VEC, int NV, bool kWarp>
static int ln_bwd_launch(const LnArgs& a, int threads, int& blocks, cudaStream_t s) {
  const long long most = ln_bwd_blocks(a.rows), need = kWarp ? (a.rows + kLnWarps - 1) / kLnWarps : a.rows;
  blocks = (int)(need < most ? need : most);
  size_t smem = sizeof(float) * a.C;
  if (kWarp && a.part) smem *= kLnWarps;   // half of the warps' two sums
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(ln_bwd_kernel<T, VEC, NV, kWarp>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024),
                            "cudaFuncSetAttribute(layernorm)"))
      return rc;
    configured[dev] = true;
  }
  return launch_kernel("ln_bwd_kernel launch", ln_bwd_kernel<T, VEC, NV, kWarp>, dim3(blocks), dim3(threads), smem, s, 1, a);
}
template <class T>
static int ln_bwd(const LnArgs& a, bool vec, int& blocks, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    const int n = a.C / V;
    if (n <= 32) return ln_bwd_launch<T, V, 1, true>(a, kLnWarps * 32, blocks, s);
    if (n <= 64) return ln_bwd_launch<T, V, 2, true>(a, kLnWarps * 32, blocks, s);
    if (n <= 96) return ln_bwd_launch<T, V, 3, true>(a, kLnWarps * 32, blocks, s);
    if (n <= 256) return ln_bwd_launch<T, V, 1, false>(a, 256, blocks, s);
    if (n <= 512) return ln_bwd_launch<T, V, 1, false>(a, 512, blocks, s);
    if (n <= 1024) return ln_bwd_launch<T, V, 2, false>(a, 512, blocks, s);
    if (n <= 2048) return ln_bwd_launch<T, V, 4, false>(a, 512, blocks, s);
  } else {
    if (a.C <= 64) return ln_bwd_launch<T, 1, 2, true>(a, kLnWarps * 32, blocks, s);
    if (a.C <= 256) return ln_bwd_launch<T, 1, 8, true>(a, kLnWarps * 32, blocks, s);
    if (a.C <= 2048) return ln_bwd_launch<T, 1, 8, false>(a, 256, blocks, s);
    if (a.C <= 8192) return ln_bwd_launch<T, 1, 8, false>(a, 1024, blocks, s);
  }
  const long long most = (long long)sm_count() * 2;
  if (int rc = launch_kernel("ln_bwd_long_kernel launch", ln_bwd_long_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(1024), 0, s, 1, a))
    return rc;
  if (!a.part) return kOk;
  const long long shares = ln_bwd_blocks(a.rows) < 64 ? ln_bwd_blocks(a.rows) : 64;
  blocks = (int)shares;
  return launch_kernel("ln_bwd_columns_kernel launch", ln_bwd_columns_kernel<T>, dim3((a.C + 255) / 256, (unsigned)shares), dim3(256), 0, s, 1, a);
}

// Whether rows of `base` can be read as 16-byte vectors.
static bool rows_of_vectors(const void* base, long long ld, int C, int bytes) {
  return al16(base) && (C * (long long)bytes) % 16 == 0 && (ld * bytes) % 16 == 0;
}

}  // namespace bxl

using namespace bxl;

extern "C" int bxl_layernorm_fwd(const void* x, long long ldx, const void* weight, const void* bias, void* y, long long ldy, float* mean,
                                 float* rstd, long long rows, int C, int dtype, int param_dtype, float eps, void* stream) {
  if (!x || !y || rows <= 0 || C <= 0) return fail(kErrInvalidArg, "bxl_layernorm_fwd: null pointer or non-positive extent (rows=%lld C=%d)", rows, C);
  if (!known_type(dtype) || (param_dtype != dtype && param_dtype != BXL_F32)) return fail(kErrUnsupported, "bxl_layernorm_fwd: weight and bias in the type of x or in fp32");
  if (C > kLnMaxC) return fail(kErrTooLarge, "bxl_layernorm_fwd: C=%d exceeds %d", C, kLnMaxC);
  if (ldx < 0 || ldy < C) return fail(kErrInvalidArg, "bxl_layernorm_fwd: bad row stride");
  if (!mean != !rstd) return fail(kErrInvalidArg, "bxl_layernorm_fwd: mean and rstd go together");
  if (!(eps >= 0.f)) return fail(kErrInvalidArg, "bxl_layernorm_fwd: eps must not be negative");
  const int b = type_bytes(dtype), pb = type_bytes(param_dtype);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % b || (reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) % pb ||
      (reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd)) % 4)
    return fail(kErrInvalidArg, "bxl_layernorm_fwd: pointers must be aligned to their elements");
  LnArgs a = {};
  a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy, a.weight = weight, a.bias = bias, a.mean = mean, a.rstd = rstd;
  a.rows = rows, a.C = C, a.param_f32 = param_dtype == BXL_F32, a.eps = eps, a.inv_c = 1.f / (float)C;
  const bool vec = rows_of_vectors(x, ldx, C, b) && rows_of_vectors(y, ldy, C, b) && al16(weight) && al16(bias);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BXL_F16) return ln_fwd<__half>(a, vec, s);
  if (dtype == BXL_BF16) return ln_fwd<__nv_bfloat16>(a, vec, s);
  return ln_fwd<float>(a, vec, s);
}

extern "C" long long bxl_layernorm_bwd_workspace_bytes(long long rows, int C) {
  if (rows <= 0 || C <= 0) return 0;
  return ln_bwd_blocks(rows) * 2ll * C * (long long)sizeof(float);
}

extern "C" int bxl_layernorm_bwd(const void* dy, long long lddy, const void* x, long long ldx, const float* mean, const float* rstd,
                                 const void* weight, void* dx, long long lddx, void* dweight, void* dbias, long long rows, int C, int dtype,
                                 int param_dtype, void* workspace, long long workspace_bytes, void* stream) {
  if (!dy || !x || !mean || !rstd || !dx || rows <= 0 || C <= 0)
    return fail(kErrInvalidArg, "bxl_layernorm_bwd: null pointer or non-positive extent (rows=%lld C=%d)", rows, C);
  if (!known_type(dtype) || (param_dtype != dtype && param_dtype != BXL_F32)) return fail(kErrUnsupported, "bxl_layernorm_bwd: weight and its gradient in the type of x or in fp32");
  if (C > kLnMaxC) return fail(kErrTooLarge, "bxl_layernorm_bwd: C=%d exceeds %d", C, kLnMaxC);
  if (ldx < 0 || lddy < 0 || lddx < C) return fail(kErrInvalidArg, "bxl_layernorm_bwd: bad row stride");
  const int b = type_bytes(dtype), pb = type_bytes(param_dtype);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx)) % b ||
      (reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(dweight) | reinterpret_cast<uintptr_t>(dbias)) % pb ||
      (reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd)) % 4)
    return fail(kErrInvalidArg, "bxl_layernorm_bwd: pointers must be aligned to their elements");
  const bool params = dweight || dbias;
  if (params) {
    if (!workspace || !al16(workspace)) return fail(kErrInvalidArg, "bxl_layernorm_bwd: workspace must be 16-byte aligned");
    if (workspace_bytes < bxl_layernorm_bwd_workspace_bytes(rows, C)) return fail(kErrTooLarge, "bxl_layernorm_bwd: workspace too small");
  }
  LnArgs a = {};
  a.x = x, a.dy = dy, a.y = dx, a.ldx = ldx, a.lddy = lddy, a.ldy = lddx, a.weight = weight;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.part = params ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows, a.C = C, a.param_f32 = param_dtype == BXL_F32, a.inv_c = 1.f / (float)C;
  const bool vec = rows_of_vectors(x, ldx, C, b) && rows_of_vectors(dy, lddy, C, b) && rows_of_vectors(dx, lddx, C, b) && al16(weight);
  cudaStream_t s = (cudaStream_t)stream;
  int blocks = 0, rc;
  if (dtype == BXL_F16) rc = ln_bwd<__half>(a, vec, blocks, s);
  else if (dtype == BXL_BF16) rc = ln_bwd<__nv_bfloat16>(a, vec, blocks, s);
  else rc = ln_bwd<float>(a, vec, blocks, s);
  if (rc || !params) return rc;
  return sum_partials(a.part, blocks, 2ll * C, C, dweight, dbias, param_dtype, s);
}
