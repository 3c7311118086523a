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
// Up to eight rows are bound by reading W once, and a tile of 128 rows by what every tile costs to set up.  Here a block forms 16
// columns: its warps share K, read W as it lies and add in shared memory.
struct FewRows {
  const void *x, *w, *bias, *residual;
  void *y, *pre;
  long long ldx, ldw, ldr, ldy, ldp;
  int M, N, K, act;
};
constexpr int kFewRows = 8, kFewColumns = 16;
// One result: `v` = x[m] . W[n].
template <class T>
__device__ __forceinline__ void few_rows_result(const FewRows& p, float v, int m, int n) {
  if (m >= p.M || n >= p.N) return;
  if (p.bias) v += to_f32(static_cast<const T*>(p.bias)[n]);
  if (p.pre) static_cast<T*>(p.pre)[m * p.ldp + n] = from_f32<T>(v);
  with_act(p.act, [&](auto act) { v = act_value<decltype(act)::value>(v); });
  if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[m * p.ldr + n]);
  static_cast<T*>(p.y)[m * p.ldy + n] = from_f32<T>(v);
}
// D[16 x 8] += A[16 x 16] B[16 x 8] of one warp
template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Rows of whole 16-byte vectors.  The warp-wide product with W as its 16-row operand and x as its 8 columns needs three
// 16-byte loads a lane for 32 values of K, and no widening: lane 4 g + q has values 8 q .. 8 q + 7 of rows g and g + 8 of W and of
// row g of x, and hands them over as the k = 2 q, 2 q + 1, 2 q + 8, 2 q + 9 of two products; both operands permute K alike.
// Bound by the loads in flight: eight rows of 2560 x 10240 (52 MB) 11.6 us, 4.5 TB/s; 1280 x 5120 5.8, 320 x 1280 2.2.  With fused
// multiply-adds instead the widening of x bounds it: 31.6, 8.9 and 3.0 us (one row of 2560 x 10240 10.5).
// Any other rows are loaded value by value, lane 4 g + q the values q, q + 4 .. q + 28, which is bound by the number of loads: 8 x 2051 x
// 8193 20.9 us, 4 x 1748 x 4672 12.3 (54.7 and 16.3 with a lane per value of K and fused multiply-adds; rows turned in shared memory 21.8
// and 10.3, but the small calls slower); 8 x 8193 x 2051 35 alone, 95 to 104 in a stream of such calls.
constexpr int kFewMaxWarps = 8;
template <class T, bool kVec>
__global__ void __launch_bounds__(kFewMaxWarps * 32) few_rows_kernel(const FewRows p) {
  pdl_launch_dependents();
  __shared__ float part[kFewMaxWarps][kFewRows * kFewColumns];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, q = lane & 3, n0 = blockIdx.x * kFewColumns;
  const T* w0 = static_cast<const T*>(p.w) + min(n0 + g, p.N - 1) * p.ldw;
  const T* w1 = static_cast<const T*>(p.w) + min(n0 + g + 8, p.N - 1) * p.ldw;
  const T* x = static_cast<const T*>(p.x) + min(g, p.M - 1) * p.ldx;
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  pdl_wait();
  auto step = [&](const uint4& a, const uint4& b, const uint4& c) {
    mma_16x8x16<T>(d, a.x, b.x, a.y, b.y, c.x, c.y);
    mma_16x8x16<T>(d, a.z, b.z, a.w, b.w, c.z, c.w);
  };
  // this lane's eight values of a row's i-th 32; behind K there are zeros
  struct Narrow {
    unsigned short v[8];
  };
  using Loaded = std::conditional_t<kVec, uint4, Narrow>;
  auto eight = [&](const T* row, int i, auto all) {
    if constexpr (kVec) {
      const int k = i * 32 + q * 8;
      return decltype(all)::value || k < p.K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
    } else {
      Narrow u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = i * 32 + 4 * j + q;
        u.v[j] = 0;
        // volatile: all of them before the first use.  (Not the read-only path: the preceding kernel may write x and W while this one's
        // blocks already wait for it.)
        if (decltype(all)::value || k < p.K) asm volatile("ld.global.u16 %0, [%1];" : "=h"(u.v[j]) : "l"(row + k));
      }
      return u;
    }
  };
  auto words = [](const Loaded& u) {
    if constexpr (kVec) return u;
    else return make_uint4(u.v[0] | u.v[1] << 16, u.v[2] | u.v[3] << 16, u.v[4] | u.v[5] << 16, u.v[6] | u.v[7] << 16);
  };
  auto take = [&](int i, auto all) {
    const Loaded a = eight(w0, i, all), b = eight(w1, i, all), c = eight(x, i, all);
    step(words(a), words(b), words(c));
  };
  constexpr int kAhead = kVec ? 4 : 2;   // twelve loads on their way at once, or 48 narrow ones
  const int whole = p.K / 32, share = (whole + warps - 1) / warps, last = min(whole, (warp + 1) * share);
  int i = warp * share;
  for (; i + kAhead <= last; i += kAhead) {
    Loaded a[kAhead], b[kAhead], c[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) a[j] = eight(w0, i + j, std::true_type{}), b[j] = eight(w1, i + j, std::true_type{}), c[j] = eight(x, i + j, std::true_type{});
#pragma unroll
    for (int j = 0; j < kAhead; ++j) step(words(a[j]), words(b[j]), words(c[j]));
  }
#pragma unroll 3
  for (; i < last; ++i) take(i, std::true_type{});
  if (warp == warps - 1 && p.K % 32) take(whole, std::false_type{});
  part[warp][2 * q * 16 + g] = d[0], part[warp][(2 * q + 1) * 16 + g] = d[1];
  part[warp][2 * q * 16 + g + 8] = d[2], part[warp][(2 * q + 1) * 16 + g + 8] = d[3];
  __syncthreads();
  for (int i = threadIdx.x; i < kFewRows * kFewColumns; i += blockDim.x) {
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += part[k][i];
    few_rows_result<T>(p, v, i / 16, n0 + i % 16);
  }
}
template <class T>
static int few_rows(const FewRows& p, bool vec, cudaStream_t s) {
  const dim3 grid((p.N + kFewColumns - 1) / kFewColumns);
  const int steps = (p.K + 31) / 32, warps = steps < kFewMaxWarps ? steps : kFewMaxWarps;
  return vec ? launch_kernel("few_rows_kernel launch", few_rows_kernel<T, true>, grid, dim3(32 * warps), 0, s, 1, p)
             : launch_kernel("few_rows_kernel launch", few_rows_kernel<T, false>, grid, dim3(32 * warps), 0, s, 1, p);
}

// ---- backward: dz and its column sums ----------------------------------------------------------
// Block (x, y): 32 * VEC columns, the y-th share of the rows, a row per warp.  Sums are taken of dz before it is rounded.
// dz is rounded to the operands' type, as PyTorch does between its own operators: the tensor cores multiply 16-bit values.  dx and dW are
// off by 1.4 times as much as with a dz kept in 32 bits (bf16 2.3e-3 for 1.7e-3 of their norm, fp16 2.9e-4 for 2.1e-4), half of
// it the rounding of the results themselves; dz in two 16-bit parts would double the work of both products.
struct DzArgs {
  const void *dy, *pre;
  void* dz;                 // null: not stored
  float* part;              // [gridDim.y][N], or null
  void* dbias;              // [N] where there is one share, or null
  long long lddy, ldp, ldz;
  int M, N, act;
};
// Few rows: one share, whose block writes the sums' result itself (32 columns and 16 warps a block, for more blocks).
constexpr int kDzRows = 2, kDzFew = 256;
template <class T, int VEC, int kDzWarps>
__global__ void __launch_bounds__(kDzWarps * 32, 32 / kDzWarps) dz_kernel(const DzArgs p) {
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
      // the rows' loads come before the first store, over which the compiler could not move them (8192 x 5120: two rows and 32 warps
      // an SM 44.7 us, four and 16 47.5, one and 48 57)
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
  if (!p.part && !p.dbias) return;
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
    if (col >= p.N) continue;
    if (p.dbias) static_cast<T*>(p.dbias)[col] = from_f32<T>(s);
    else p.part[blockIdx.y * (long long)p.N + col] = s;
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
  if (M <= kDzFew) return 1;
  const long long cols = (N + 32ll * vec - 1) / (32 * vec);
  long long shares = (sm_count() * 8ll + cols - 1) / cols;
  const long long most = ((long long)M + 31) / 32;
  if (shares > most) shares = most;
  return shares < 1 ? 1 : shares > 4096 ? 4096 : (int)shares;
}

// The partial sums of dbias: room for the vector form, which has more shares than the other.
static long long dbias_part_bytes(const bxl_linear_args* a) { return a->dbias && a->M > kDzFew ? 4ll * dz_shares(a->M, a->N, 8) * a->N : 0; }

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

// z = x W^T, before the operands' places are known
static LinearProduct forward_product(const bxl_linear_args* a) {
  LinearProduct q = {};
  q.bf16 = a->dtype == BXL_BF16, q.bias = a->bias, q.residual = a->residual, q.ldr = a->ldr, q.C = a->y, q.ldc = a->ldy, q.pre = a->pre, q.ldp = a->ldp;
  q.act = a->act, q.M = a->M, q.N = a->N, q.K = a->K;
  return q;
}
// dx[M,K] = dz[M,N] W[N,K]
static LinearProduct x_grad_product(const bxl_linear_args* a) {
  LinearProduct q = {};
  q.bf16 = a->dtype == BXL_BF16, q.b_kn = 1, q.C = a->dx, q.ldc = a->lddx, q.M = a->M, q.N = a->K, q.K = a->N;
  return q;
}
// dW[N,K] = dz^T[N,M] x[M,K]
static LinearProduct w_grad_product(const bxl_linear_args* a) {
  LinearProduct q = {};
  q.bf16 = a->dtype == BXL_BF16, q.a_mn = 1, q.b_kn = 1, q.C = a->dweight, q.ldc = a->lddw, q.M = a->N, q.N = a->K, q.K = a->M;
  return q;
}
static long long fwd_workspace(const bxl_linear_args* a) {
  if (a->M <= kFewRows) return 0;
  const LinearProduct q = forward_product(a), *one = &q;
  return round256(copy_bytes(a->x, a->ldx, a->M, a->K)) + round256(copy_bytes(a->weight, a->ldw, a->N, a->K)) + linear_workspace(&one, 1);
}
// dz is dy itself where there is no activation and the copy engine can read it
static bool stores_dz(const bxl_linear_args* a) {
  return (a->dx || a->dweight) && (a->act != BXL_ACT_NONE || !tma_rows(a->dy, a->lddy, a->N));
}
static long long bwd_workspace(const bxl_linear_args* a) {
  long long n = 0;
  if (stores_dz(a)) n += round256(2ll * a->M * round8(a->N));
  n += round256(dbias_part_bytes(a));
  if (a->dx) n += round256(copy_bytes(a->weight, a->ldw, a->N, a->K));
  if (a->dweight) n += round256(copy_bytes(a->x, a->ldx, a->M, a->K));
  const LinearProduct x = x_grad_product(a), w = w_grad_product(a);
  const LinearProduct* q[2] = {a->dx ? &x : &w, &w};
  if (a->dx || a->dweight) n += linear_workspace(q, a->dx && a->dweight ? 2 : 1);
  return n;
}

}  // namespace bxl

using namespace bxl;

extern "C" long long bxl_linear_act_fwd_workspace_bytes(const bxl_linear_args* a) { return check_linear("bxl_linear_act_fwd", a) ? 0 : fwd_workspace(a); }

extern "C" int bxl_linear_act_fwd(const bxl_linear_args* a, int* launches, void* stream) {
  const char* who = "bxl_linear_act_fwd";
  if (int rc = check_linear(who, a)) return rc;
  if (!a->y) return fail(kErrInvalidArg, "%s: null operand", who);
  if (a->ldy < a->N || (a->pre && a->ldp < a->N) || (a->residual && a->ldr < 0)) return fail(kErrInvalidArg, "%s: bad leading dimension", who);
  if (int rc = check_workspace(who, a, fwd_workspace(a))) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int bf16 = a->dtype == BXL_BF16;
  int count = 0;
  if (launches) *launches = 1;
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
  LinearProduct q = forward_product(a);
  const LinearProduct* one = &q;
  q.A = x.dst ? x.dst : x.src, q.lda = x.ld_dst, q.B = w.dst ? w.dst : w.src, q.ldb = w.ld_dst, q.b_is_weight = !w.dst;
  if (x.dst || w.dst) ++count;
  if (int rc = linear_products(&one, 1, ws.at, &count, s)) return rc;
  if (launches) *launches = count;
  return kOk;
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
    const bool few = a->M <= kDzFew;
    const bool vec = !few && a->N % 8 == 0 && al(a->dy, 16) && a->lddy % 8 == 0 && (a->act == BXL_ACT_NONE || (al(a->pre, 16) && a->ldp % 8 == 0));
    const int shares = dz_shares(a->M, a->N, vec ? 8 : 1), cols = vec ? 256 : 32;
    if (a->dbias && few) p.dbias = a->dbias;
    else if (a->dbias) p.part = static_cast<float*>(ws.take(dbias_part_bytes(a)));
    const dim3 grid((a->N + cols - 1) / cols, shares);
    auto launch = [&](auto kernel, int warps) { return launch_kernel("dz_kernel launch", kernel, grid, dim3(32 * warps), 0, s, 1, p); };
    int rc;
    if (bf16) rc = few ? launch(dz_kernel<__nv_bfloat16, 1, 16>, 16) : vec ? launch(dz_kernel<__nv_bfloat16, 8, 8>, 8) : launch(dz_kernel<__nv_bfloat16, 1, 8>, 8);
    else rc = few ? launch(dz_kernel<__half, 1, 16>, 16) : vec ? launch(dz_kernel<__half, 8, 8>, 8) : launch(dz_kernel<__half, 1, 8>, 8);
    if (rc) return rc;
    ++count;
    if (p.part) {
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
  LinearProduct x_grad = x_grad_product(a), w_grad = w_grad_product(a);
  x_grad.A = dz, x_grad.lda = ldz, x_grad.B = w.dst ? w.dst : w.src, x_grad.ldb = w.ld_dst, x_grad.b_is_weight = !w.dst;
  w_grad.A = dz, w_grad.lda = ldz, w_grad.B = x.dst ? x.dst : x.src, w_grad.ldb = x.ld_dst;
  const LinearProduct* q[2] = {a->dx ? &x_grad : &w_grad, &w_grad};
  if (a->dx || a->dweight)
    if (int rc = linear_products(q, a->dx && a->dweight ? 2 : 1, ws.at, &count, s)) return rc;
  if (launches) *launches = count;
  return kOk;
}
