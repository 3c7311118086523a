// Linear layers with bias, activation and residual, forward and backward, fp16 or bf16.
//
//   forward    z = x W^T + b,  y = act(z) + residual
//   backward   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// The products run on the tensor cores (linear_product in gemm_conv.cu), with everything else of the forward pass in their
// epilogue; W and x are read as they lie (K-major or MN-major operands), dW takes dz transposed in the same way.  Here are
// the kernels around them: the product of a few rows, bound by reading W once, and the pass that forms dz and its column sums,
// bound by memory.
#include "bxl_act.cuh"
#include "bxl_common.cuh"
#include "bxl_host.h"
#include "bxl_types.cuh"

namespace bxl {

// ---- forward of a few rows -------------------------------------------------------------------
// A warp forms NB neighbouring columns of all MB rows over its share of K: every 16 bytes of W are loaded once, by one
// lane, and meet the same 16 bytes of K of every row of x (from L1).  The block's warps share K and add in shared memory.
struct FewRows {
  const void *x, *w, *bias, *residual;
  void *y, *pre;
  long long ldx, ldw, ldr, ldy, ldp;
  int M, N, K, act;
};
template <class T, int VEC, int MB, int NB>
__global__ void __launch_bounds__(256) few_rows_kernel(const FewRows p) {
  static_assert(MB * NB <= 32, "one lane per result");
  pdl_launch_dependents();
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int n0 = blockIdx.x * NB;
  const T* x = static_cast<const T*>(p.x);
  const T* w[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) w[j] = static_cast<const T*>(p.w) + (long long)min(n0 + j, p.N - 1) * p.ldw;
  float acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = 0.f;
  pdl_wait();
  const int vecs = p.K / VEC;
#pragma unroll 2
  for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
    Vec<T, VEC> wv[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) wv[j] = load_vec<T, VEC>(w[j] + (long long)v * VEC);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const Vec<T, VEC> xv = load_vec<T, VEC>(x + min(i, p.M - 1) * p.ldx + (long long)v * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = fmaf(to_f32(xv.v[e]), to_f32(wv[j].v[e]), acc[i][j]);
    }
  }
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float s = acc[i][j];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == i * NB + j) mine = s;
    }
  if (warps > 1) {
    part[warp][lane] = mine;
    __syncthreads();
    if (warp) return;
    for (int k = 1; k < warps; ++k) mine += part[k][lane];
  }
  const int m = lane / NB, n = n0 + lane % NB;
  if (lane >= MB * NB || m >= p.M || n >= p.N) return;
  if (p.bias) mine += to_f32(static_cast<const T*>(p.bias)[n]);
  if (p.pre) static_cast<T*>(p.pre)[m * p.ldp + n] = from_f32<T>(mine);
  with_act(p.act, [&](auto act) { mine = act_value<decltype(act)::value>(mine); });
  if (p.residual) mine += to_f32(static_cast<const T*>(p.residual)[m * p.ldr + n]);
  static_cast<T*>(p.y)[m * p.ldy + n] = from_f32<T>(mine);
}

constexpr int kFewRows = 8;
template <class T, int VEC, int MB>
static int few_rows_launch(const FewRows& p, cudaStream_t s) {
  constexpr int NB = 4;
  const int groups = (p.N + NB - 1) / NB, most = (p.K / VEC + 31) / 32;
  int warps = (sm_count() * 8 + groups - 1) / groups;   // eight warps an SM, as long as each has a vector per lane
  warps = warps > most ? most : warps;
  warps = warps > 8 ? 8 : warps < 1 ? 1 : warps;
  return launch_kernel("few_rows_kernel launch", few_rows_kernel<T, VEC, MB, NB>, dim3(groups), dim3(32 * warps), 0, s, 1, p);
}
template <class T>
static int few_rows(const FewRows& p, bool vec, cudaStream_t s) {
  if (p.M == 1) return vec ? few_rows_launch<T, 8, 1>(p, s) : few_rows_launch<T, 1, 1>(p, s);
  if (p.M == 2) return vec ? few_rows_launch<T, 8, 2>(p, s) : few_rows_launch<T, 1, 2>(p, s);
  if (p.M <= 4) return vec ? few_rows_launch<T, 8, 4>(p, s) : few_rows_launch<T, 1, 4>(p, s);
  return vec ? few_rows_launch<T, 8, 8>(p, s) : few_rows_launch<T, 1, 8>(p, s);
}

// ---- backward: dz and its column sums ----------------------------------------------------------
// Block (x, y): 32 * VEC columns, the y-th share of the rows, a row per warp.  Sums are taken of dz before it is rounded.
struct DzArgs {
  const void *dy, *pre;
  void* dz;                 // null: not stored
  float* part;              // [gridDim.y][N], or null
  long long lddy, ldp, ldz;
  int M, N, act;
};
constexpr int kDzWarps = 8, kDzRows = 4;
template <class T, int VEC>
__global__ void __launch_bounds__(kDzWarps * 32) dz_kernel(const DzArgs p) {
  pdl_launch_dependents();
  using F = typename Lanes<VEC>::F;
  constexpr int N = Lanes<VEC>::N;
  __shared__ float sums[kDzWarps][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * VEC;
  const int per = (p.M + gridDim.y - 1) / gridDim.y;
  const long long r1 = min((long long)p.M, (blockIdx.y + 1ll) * per);
  F acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = splat<F>(0.f);
  pdl_wait();
  if (c < p.N)
    with_act(p.act, [&](auto act) {
      constexpr int kAct = decltype(act)::value;
      // four rows are loaded before the first result is stored: the compiler cannot move loads over stores
      for (long long r0 = (long long)blockIdx.y * per + warp; r0 < r1; r0 += kDzRows * kDzWarps) {
        Vec<T, VEC> g[kDzRows], z[kDzRows];
#pragma unroll
        for (int i = 0; i < kDzRows; ++i) {
          const long long r = r0 + i * kDzWarps;
          if (r < r1) {
            g[i] = load_vec<T, VEC>(static_cast<const T*>(p.dy) + r * p.lddy + c);
            if constexpr (kAct != BXL_ACT_NONE) z[i] = load_vec<T, VEC>(static_cast<const T*>(p.pre) + r * p.ldp + c);
          }
        }
#pragma unroll
        for (int i = 0; i < kDzRows; ++i) {
          const long long r = r0 + i * kDzWarps;
          if (r >= r1) break;
          F d[N];
          widen<T, VEC>(g[i], d);
          if constexpr (kAct != BXL_ACT_NONE) {
            F u[N];
            widen<T, VEC>(z[i], u);
#pragma unroll
            for (int j = 0; j < N; ++j) d[j] = mul(d[j], act_slope<kAct>(u[j]));
          }
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] = add(acc[j], d[j]);
          if (p.dz) store_vec<T, VEC>(static_cast<T*>(p.dz) + r * p.ldz + c, narrow<T, VEC>(d));
        }
      }
    });
  if (!p.part) return;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (VEC == 1) {
      sums[warp][lane] = acc[j];
    } else {
      const float2 u = split(acc[j]);
      sums[warp][lane + 64 * j] = u.x, sums[warp][lane + 64 * j + 32] = u.y;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += kDzWarps * 32) {
    const int col = (blockIdx.x * 32 + i % 32) * VEC + i / 32;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kDzWarps; ++w) s += sums[w][i];
    if (col < p.N) p.part[blockIdx.y * (long long)p.N + col] = s;
  }
}

// ---- host side -----------------------------------------------------------------------------------
static bool al(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
static long long round8(long long n) { return (n + 7) / 8 * 8; }
// Whether the copy engine can read these rows as they are.
static bool tma_rows(const void* p, long long ld, int cols) { return al(p, 16) && ld % 8 == 0 && ld >= cols; }
static long long copy_bytes(const void* p, long long ld, int rows, int cols) { return tma_rows(p, ld, cols) ? 0 : 2ll * rows * round8(cols); }
static long long round256(long long n) { return (n + 255) / 256 * 256; }

// Shares of the rows in dz_kernel: about eight blocks an SM, and at least 32 rows each.
static int dz_shares(int M, int N, int vec) {
  const long long cols = (N + 32ll * vec - 1) / (32 * vec);
  long long shares = (sm_count() * 8ll + cols - 1) / cols;
  const long long most = ((long long)M + 31) / 32;
  if (shares > most) shares = most;
  return shares < 1 ? 1 : shares > 4096 ? 4096 : (int)shares;
}

static int check_linear(const char* who, const bxl_linear_args* a) {
  if (!a) return fail(kErrInvalidArg, "%s: null argument block", who);
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return fail(kErrInvalidArg, "%s: non-positive extent M=%d N=%d K=%d", who, a->M, a->N, a->K);
  if (a->M > (1 << 30) || a->N > (1 << 30) || a->K > (1 << 30)) return fail(kErrTooLarge, "%s: extents of at most 2^30", who);
  if (a->dtype != BXL_F16 && a->dtype != BXL_BF16) return fail(kErrUnsupported, "%s: fp16 or bf16", who);
  if (a->act < BXL_ACT_NONE || a->act > BXL_ACT_QUICK_GELU) return fail(kErrUnsupported, "%s: unknown activation %d", who, a->act);
  const void* all[] = {a->x, a->weight, a->bias, a->residual, a->y, a->pre, a->dy, a->dx, a->dweight, a->dbias};
  for (const void* p : all)
    if (!al(p, 2)) return fail(kErrInvalidArg, "%s: operands must be 2-byte aligned", who);
  if (!a->x || !a->weight) return fail(kErrInvalidArg, "%s: null operand", who);
  if (a->ldx < 0 || a->ldw < 0) return fail(kErrInvalidArg, "%s: bad leading dimension", who);
  return kOk;
}

struct Workspace {
  char* at;
  void* take(long long bytes) {
    void* p = at;
    at += round256(bytes);
    return p;
  }
};
static int check_workspace(const char* who, const bxl_linear_args* a, long long need) {
  if (need <= 0) return kOk;
  if (!a->workspace || !al(a->workspace, 16)) return fail(kErrInvalidArg, "%s: workspace must be 16-byte aligned", who);
  if (a->workspace_bytes < need) return fail(kErrTooLarge, "%s: workspace too small", who);
  return kOk;
}

static long long fwd_workspace(const bxl_linear_args* a) {
  if (a->M <= kFewRows) return 0;
  return round256(copy_bytes(a->x, a->ldx, a->M, a->K)) + round256(copy_bytes(a->weight, a->ldw, a->N, a->K));
}
// dz is dy itself where there is no activation and the copy engine can read it
static bool stores_dz(const bxl_linear_args* a) {
  return (a->dx || a->dweight) && (a->act != BXL_ACT_NONE || !tma_rows(a->dy, a->lddy, a->N));
}
static long long bwd_workspace(const bxl_linear_args* a) {
  long long n = 0;
  if (stores_dz(a)) n += round256(2ll * a->M * round8(a->N));
  if (a->dbias) n += round256(4ll * dz_shares(a->M, a->N, 1) * a->N);
  if (a->dx) n += round256(copy_bytes(a->weight, a->ldw, a->N, a->K));
  if (a->dweight) n += round256(copy_bytes(a->x, a->ldx, a->M, a->K));
  return n;
}

}  // namespace bxl

using namespace bxl;

extern "C" long long bxl_linear_act_fwd_workspace_bytes(const bxl_linear_args* a) { return check_linear("bxl_linear_act_fwd", a) ? 0 : fwd_workspace(a); }

extern "C" int bxl_linear_act_fwd(const bxl_linear_args* a, void* stream) {
  const char* who = "bxl_linear_act_fwd";
  if (int rc = check_linear(who, a)) return rc;
  if (!a->y) return fail(kErrInvalidArg, "%s: null operand", who);
  if (a->ldy < a->N || (a->pre && a->ldp < a->N) || (a->residual && a->ldr < 0)) return fail(kErrInvalidArg, "%s: bad leading dimension", who);
  if (int rc = check_workspace(who, a, fwd_workspace(a))) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int bf16 = a->dtype == BXL_BF16;
  if (a->M <= kFewRows) {
    const FewRows p{a->x, a->weight, a->bias, a->residual, a->y, a->pre, a->ldx, a->ldw, a->ldr, a->ldy, a->ldp, a->M, a->N, a->K, a->act};
    const bool vec = a->K % 8 == 0 && al(a->x, 16) && al(a->weight, 16) && a->ldx % 8 == 0 && a->ldw % 8 == 0;
    return bf16 ? few_rows<__nv_bfloat16>(p, vec, s) : few_rows<__half>(p, vec, s);
  }
  Workspace ws{static_cast<char*>(a->workspace)};
  RowCopy x{a->x, nullptr, a->ldx, a->ldx, a->M, a->K}, w{a->weight, nullptr, a->ldw, a->ldw, a->N, a->K};
  if (const long long n = copy_bytes(a->x, a->ldx, a->M, a->K)) x.dst = ws.take(n), x.ld_dst = round8(a->K);
  if (const long long n = copy_bytes(a->weight, a->ldw, a->N, a->K)) w.dst = ws.take(n), w.ld_dst = round8(a->K);
  if (int rc = repack_rows(x, w, s)) return rc;
  LinearProduct q = {};
  q.A = x.dst ? x.dst : x.src, q.lda = x.ld_dst, q.B = w.dst ? w.dst : w.src, q.ldb = w.ld_dst, q.b_is_weight = !w.dst;
  q.bias = a->bias, q.residual = a->residual, q.ldr = a->ldr, q.C = a->y, q.ldc = a->ldy, q.pre = a->pre, q.ldp = a->ldp;
  q.act = a->act, q.bf16 = bf16, q.M = a->M, q.N = a->N, q.K = a->K;
  return linear_product(q, s);
}

extern "C" long long bxl_linear_act_bwd_workspace_bytes(const bxl_linear_args* a) { return check_linear("bxl_linear_act_bwd", a) ? 0 : bwd_workspace(a); }

extern "C" int bxl_linear_act_bwd(const bxl_linear_args* a, int* launches, void* stream) {
  const char* who = "bxl_linear_act_bwd";
  if (int rc = check_linear(who, a)) return rc;
  if (!a->dy || (a->act != BXL_ACT_NONE && !a->pre)) return fail(kErrInvalidArg, "%s: dy, and with an activation the value before it, are needed", who);
  if (a->lddy < 0 || (a->pre && a->ldp < 0) || (a->dx && a->lddx < a->K) || (a->dweight && a->lddw < a->K))
    return fail(kErrInvalidArg, "%s: bad leading dimension", who);
  if (int rc = check_workspace(who, a, bwd_workspace(a))) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int bf16 = a->dtype == BXL_BF16;
  int count = 0;
  Workspace ws{static_cast<char*>(a->workspace)};
  const void* dz = a->dy;
  long long ldz = a->lddy;
  if (stores_dz(a) || a->dbias) {
    DzArgs p = {};
    p.dy = a->dy, p.lddy = a->lddy, p.pre = a->pre, p.ldp = a->ldp, p.M = a->M, p.N = a->N, p.act = a->act;
    if (stores_dz(a)) {
      ldz = p.ldz = round8(a->N);
      dz = p.dz = ws.take(2ll * a->M * ldz);
    }
    const bool vec = a->N % 8 == 0 && al(a->dy, 16) && a->lddy % 8 == 0 && (a->act == BXL_ACT_NONE || (al(a->pre, 16) && a->ldp % 8 == 0));
    const int shares = dz_shares(a->M, a->N, vec ? 8 : 1), cols = vec ? 256 : 32;
    if (a->dbias) p.part = static_cast<float*>(ws.take(4ll * dz_shares(a->M, a->N, 1) * a->N));
    const dim3 grid((a->N + cols - 1) / cols, shares), block(kDzWarps * 32);
    int rc;
    if (bf16) rc = vec ? launch_kernel("dz_kernel launch", dz_kernel<__nv_bfloat16, 8>, grid, block, 0, s, 1, p) : launch_kernel("dz_kernel launch", dz_kernel<__nv_bfloat16, 1>, grid, block, 0, s, 1, p);
    else rc = vec ? launch_kernel("dz_kernel launch", dz_kernel<__half, 8>, grid, block, 0, s, 1, p) : launch_kernel("dz_kernel launch", dz_kernel<__half, 1>, grid, block, 0, s, 1, p);
    if (rc) return rc;
    ++count;
    if (a->dbias) {
      if (int r = sum_partials(p.part, shares, a->N, a->N, a->dbias, nullptr, a->dtype, s)) return r;
      ++count;
    }
  }
  RowCopy x{a->x, nullptr, a->ldx, a->ldx, a->M, a->K}, w{a->weight, nullptr, a->ldw, a->ldw, a->N, a->K};
  if (a->dx)
    if (const long long n = copy_bytes(a->weight, a->ldw, a->N, a->K)) w.dst = ws.take(n), w.ld_dst = round8(a->K);
  if (a->dweight)
    if (const long long n = copy_bytes(a->x, a->ldx, a->M, a->K)) x.dst = ws.take(n), x.ld_dst = round8(a->K);
  if (x.dst || w.dst) {
    if (int rc = repack_rows(x, w, s)) return rc;
    ++count;
  }
  LinearProduct q = {};
  q.bf16 = bf16;
  if (a->dx) {
    // dx[M,K] = dz[M,N] W[N,K]
    q.A = dz, q.lda = ldz, q.a_mn = 0, q.B = w.dst ? w.dst : w.src, q.ldb = w.ld_dst, q.b_kn = 1, q.b_is_weight = !w.dst;
    q.C = a->dx, q.ldc = a->lddx, q.M = a->M, q.N = a->K, q.K = a->N;
    if (int rc = linear_product(q, s)) return rc;
    ++count;
  }
  if (a->dweight) {
    // dW[N,K] = dz^T[N,M] x[M,K]
    q.A = dz, q.lda = ldz, q.a_mn = 1, q.B = x.dst ? x.dst : x.src, q.ldb = x.ld_dst, q.b_kn = 1, q.b_is_weight = 0;
    q.C = a->dweight, q.ldc = a->lddw, q.M = a->N, q.N = a->K, q.K = a->M;
    if (int rc = linear_product(q, s)) return rc;
    ++count;
  }
  if (launches) *launches = count;
  return kOk;
}
