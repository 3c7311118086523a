// LayerNorm over the last axis, forward and backward, fp16 / bf16 / fp32 rows of any length.
//
//   forward   m = sum(x) / C,  r = 1 / sqrt(sum((x - m)^2) / C + eps),  y = (x - m) r w + b
//   backward  h = (x - m) r,  g = dy w:  dx = r (g - mean(g) - h mean(g h)),
//             dw = sum over rows of dy h,  db = sum over rows of dy
//
// Memory bounds it in principle: the forward pass reads x and writes y once, the backward pass reads dy and x and writes dx
// once.  At 8 bytes a cycle and SM and 16-bit values that leaves some 20 (forward) and 30 (backward) instructions for a
// value, so issue slots come close: arithmetic is on pairs (F2), and a value is widened once and kept.  Sums are fp32; the
// variance is taken of the differences from the mean.  dw and db: every thread keeps the sums of its own columns over
// all rows that it meets, a block adds those of its threads, and a second launch adds the blocks' in a fixed order (no
// atomics).
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
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  if (warps > 4) return warp_sum(lane < warps ? slot[lane] : 0.f);
  v = slot[0];
  for (int i = 1; i < warps; ++i) v += slot[i];
  return v;
}
// Sum over LANES neighbouring lanes (8, 16 or 32), or over the block (0).
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  if constexpr (LANES == 0) {
    return block_sum(v, slot);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
}

// ---- forward: a row in registers -------------------------------------------------------------
// LANES lanes per row (0: a block per row), NV vectors of VEC elements each.  The next row is on its way while the present
// one is reduced.
constexpr int kLnWarps = 8;   // warps of a block that holds several rows
template <class T, int VEC, int NV, int LANES, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) ln_fwd_kernel(const LnArgs a) {
  pdl_launch_dependents();
  using F = typename Lanes<VEC>::F;
  constexpr int N = Lanes<VEC>::N;
  __shared__ float red[2][32];
  constexpr int kRows = LANES ? kLnWarps * 32 / LANES : 1;   // rows of a block
  constexpr int kTogether = LANES ? 32 / LANES : 1;          // rows of a warp
  const int tid = LANES ? threadIdx.x % LANES : threadIdx.x;
  const int step = LANES ? LANES : blockDim.x;
  const int n = a.C / VEC;
  const Param<T> w{a.weight, a.param_f32}, b{a.bias, a.param_f32};
  const long long stride = gridDim.x * (long long)kRows;
  long long r = blockIdx.x * (long long)kRows + (LANES ? threadIdx.x / LANES : 0);
  Vec<T, VEC> next[NV];
  auto fetch = [&](long long row) {
    if (row >= a.rows) return;
    const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) next[i] = load_vec<T, VEC>(xr + (tid + i * step) * VEC);
  };
  pdl_wait();
  fetch(r);
  // the lanes of a warp stay together: those of rows past the last one take part in the sums
  const long long last = (a.rows + kTogether - 1) / kTogether * kTogether;
  for (; r < last; r += stride) {
    F x[NV][N];
    F s = splat<F>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
        widen<T, VEC>(next[i], x[i]);
#pragma unroll
        for (int j = 0; j < N; ++j) s = add(s, x[i][j]);
      }
    fetch(r + stride);
    const float mean = row_sum<LANES>(total(s), red[0]) / a.C;   // a division: the mean of equal values is their value
    const F minus = splat<F>(-mean);
    F q = splat<F>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * step < n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          x[i][j] = add(x[i][j], minus);
          q = fma(x[i][j], x[i][j], q);
        }
      }
    const float rstd = rsqrtf(row_sum<LANES>(total(q), red[1]) * a.inv_c + a.eps);
    if (r < a.rows) {
      T* yr = static_cast<T*>(a.y) + r * a.ldy;
      const F scale = splat<F>(rstd);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * step) * VEC;
        if (tid + i * step < n) {
          F wv[N], bv[N];
          w.template get<VEC>(c, 1.f, wv);
          b.template get<VEC>(c, 0.f, bv);
#pragma unroll
          for (int j = 0; j < N; ++j) x[i][j] = fma(mul(x[i][j], scale), wv[j], bv[j]);
          store_vec<T, VEC>(yr + c, narrow<T, VEC>(x[i]));
        }
      }
      if (a.mean && tid == 0) a.mean[r] = mean, a.rstd[r] = rstd;
    }
  }
}

// Rows of any length that nothing else takes: three passes over the row, the second and third mostly from L2.
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

// ---- many rows: teams ------------------------------------------------------------------------
// A team of TL threads (8 to a whole block) takes one row at a time and keeps it in registers between its sums and its result;
// thread `i` of a team has the columns i, i + TL, ... of every row, so that the parameters (forward) and the column sums
// (backward) stay in registers over all rows.  Rows come through a ring of stages of their own per team, filled by the bulk
// copy engine: the bytes in flight depend neither on registers nor on occupancy.  Teams below a warp share the warp's stage.
//
// Rows of whole 16-byte vectors are copied one by one.  Rows of other lengths can be copied where they lie back to back from an
// aligned address on: the span is then widened to 16-byte boundaries (what it touches beside the row belongs to its
// neighbours), and what lies behind the tensor's last boundary is copied by hand.
struct LnTeams {
  int TL, stages;           // threads of a team; copies in flight of a ring
  int per, groups, rows;    // rows that a warp has at a time; how often in a unit; the unit's rows
  uint32_t units;           // a.rows in steps of `rows`
  int one_copy;             // a unit's rows lie back to back
  int mat_bytes;            // a stage's room for one matrix
  unsigned long long ceiling;    // elements of x and dy before their last 16-byte boundary
  int off_w, off_red, off_bar;   // shared-memory offsets: weight, partial sums, barriers (the rings come first)
  int* dev_status;
};
constexpr int kTeamThreads = 512, kTeamWarps = kTeamThreads / 32;
// Teams of several warps; of a warp or less (kSub below); of a warp or less with several rows of each team in a unit.
enum { kWide, kNarrow, kGrouped };

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Where a stage's first element lies in its room.
template <class T, int VEC>
__device__ __forceinline__ uint32_t stage_shift(uint32_t row0, int C) {
  return VEC == 1 ? (row0 * static_cast<uint32_t>(C)) & (16 / sizeof(T) - 1) : 0;
}
// Called by all lanes of one warp: rows [row0, row0 + n) of the given matrices, each to its room of the stage.
template <class T, int VEC, int MATS>
__device__ __forceinline__ void load_stage(const T* const (&src)[MATS], const long long (&ld)[MATS], const LnArgs& a, const LnTeams& t, uint32_t row0, int n,
                                           uint8_t* stage, uint32_t bar) {
  const int lane = threadIdx.x & 31;
  if constexpr (VEC == 1) {
    constexpr unsigned long long kUnit = 16 / sizeof(T);
    if (lane == 0) {
      const unsigned long long begin = static_cast<unsigned long long>(row0) * a.C, first = begin & ~(kUnit - 1), end = begin + static_cast<uint32_t>(n * a.C);
      unsigned long long stop = (end + kUnit - 1) & ~(kUnit - 1);
      if (stop > t.ceiling) {
        stop = t.ceiling > first ? t.ceiling : first;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
          for (unsigned long long i = stop; i < end; ++i) reinterpret_cast<T*>(stage + m * t.mat_bytes)[i - first] = src[m][i];
      }
      const uint32_t bytes = static_cast<uint32_t>(stop - first) * sizeof(T);
      mbar_arrive_expect_tx(bar, MATS * bytes);
      if (bytes) {
#pragma unroll
        for (int m = 0; m < MATS; ++m) bulk_load(smem_u32(stage + m * t.mat_bytes), src[m] + first, bytes, bar);
      }
    }
  } else {
    const uint32_t row_bytes = a.C * sizeof(T);
    if (t.one_copy) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, MATS * n * row_bytes);
#pragma unroll
        for (int m = 0; m < MATS; ++m) bulk_load(smem_u32(stage + m * t.mat_bytes), src[m] + row0 * ld[m], n * row_bytes, bar);
      }
    } else {
      if (lane == 0) mbar_arrive_expect_tx(bar, MATS * n * row_bytes);
      __syncwarp();
      if (lane < n) {
#pragma unroll
        for (int m = 0; m < MATS; ++m) bulk_load(smem_u32(stage + m * t.mat_bytes) + lane * row_bytes, src[m] + (row0 + lane) * ld[m], row_bytes, bar);
      }
    }
  }
}
// After a wait that gave up: copies that may still be in flight land before the block's shared memory is released.
__device__ __forceinline__ void let_copies_land() {
  const unsigned long long t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
}
// Barrier of the `threads` threads of one team; whether any of them raised `flag`.
__device__ __forceinline__ bool team_barrier(int id, int threads, bool flag) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(flag))
      : "memory");
  return any != 0;
}
// What a thread is in its team.
struct TeamRole {
  int lane;                // in the team
  int warps, warp;         // warps of the team, and which of them
  int team, teams;         // of the block (a warp's teams count as one)
  int sub;                 // which of a warp's rows
  __device__ __forceinline__ explicit TeamRole(int TL) {
    lane = threadIdx.x % TL;
    warps = TL > 32 ? TL / 32 : 1, warp = threadIdx.x / 32 % warps;
    team = threadIdx.x / (32 * warps), teams = kTeamWarps / warps;
    sub = TL < 32 ? (threadIdx.x & 31) / TL : 0;
  }
};
// Sums over a team of two values at once.  Teams of several warps meet at a barrier, once: partial sums take turns between
// two slots.  Returns whether a wait has failed.
template <int K>
__device__ __forceinline__ void add_lanes(float (&v)[K], int o) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
}
template <int K, bool kSub>
__device__ __forceinline__ bool team_sum(float (&v)[K], const LnTeams& t, const TeamRole& me, float* slots, int turn, bool failed) {
  if (!kSub || t.TL > 16) add_lanes<K>(v, 16);
  if (!kSub || t.TL > 8) add_lanes<K>(v, 8);
  add_lanes<K>(v, 4);
  add_lanes<K>(v, 2);
  add_lanes<K>(v, 1);
  if constexpr (kSub) return failed;
  float* s = slots + (me.team * 2 + turn) * me.warps * K;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) s[me.warp * K + k] = v[k];
  }
  failed = team_barrier(1 + me.team, 32 * me.warps, failed);
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = s[(threadIdx.x & (me.warps - 1)) * K + k];
  if (me.warps > 8) add_lanes<K>(v, 8);
  if (me.warps > 4) add_lanes<K>(v, 4);
  if (me.warps > 2) add_lanes<K>(v, 2);
  add_lanes<K>(v, 1);
  return failed;
}
// s / C, exact where the quotient is (equal values have that value as their mean): a product and one correction, which an infinite sum
// does without.
__device__ __forceinline__ float mean_of(float s, const LnArgs& a) {
  const float m = s * a.inv_c;
  const float exact = fmaf(fmaf(-m, static_cast<float>(a.C), s), a.inv_c, m);
  return fabsf(m) < INFINITY ? exact : m;
}
// A vector of fp32 parameters in shared memory: quarters of 16 bytes of neighbouring vectors lie side by side (two
// planes for VEC = 8), so that a warp's reads meet no bank twice.
template <int VEC>
__device__ __forceinline__ void shared_param(const float* s, int n, int v, typename Lanes<VEC>::F (&out)[Lanes<VEC>::N]) {
  if constexpr (VEC == 1) {
    out[0] = s[v];
  } else {
#pragma unroll
    for (int q = 0; q < VEC / 4; ++q) {
      const float4 u = *reinterpret_cast<const float4*>(s + (q * n + v) * 4);
      out[2 * q] = f2(u.x, u.y), out[2 * q + 1] = f2(u.z, u.w);
    }
  }
}
template <int VEC>
__device__ __forceinline__ int shared_param_index(int n, int c) {
  if constexpr (VEC == 1) return c;
  else return ((c % VEC / 4) * n + c / VEC) * 4 + c % 4;
}
// Which of a thread's NV vectors may lie behind the row's end: the host picks NV so that only the last one does (the last four
// single elements).
template <int VEC, int NV>
__device__ __forceinline__ bool has_vector(int i, int v, int n) {
  return i < NV - (VEC == 1 ? 4 : 1) || v < n;
}

// The ring of a team: what its first warp fills and all of it waits on.  Rows are counted in 32 bits (the products and comparisons
// of 64 were a fifth of the instructions of narrow rows), and little is kept between units: registers bound the backward kernel.
template <class T, int VEC, int MATS, bool kSub>
struct TeamRing {
  const LnArgs& a;
  const LnTeams& t;
  uint8_t* base;
  uint32_t bars;
  volatile int* abort_flag;
  uint32_t row, step;       // the unit's first row; rows that the grid's teams take at a time
  int left, last_n;         // units of this team still to come, this one included; rows of its last one
  int stage;
  uint32_t phase;
  __device__ __forceinline__ TeamRing(const LnArgs& a_, const LnTeams& t_, uint8_t* smem, const TeamRole& me) : a(a_), t(t_) {
    const uint32_t first = blockIdx.x * me.teams + me.team, units = gridDim.x * me.teams, rows = kSub ? t.rows : 1;
    row = first * rows, step = units * rows;
    left = first < t.units ? static_cast<int>((t.units - 1 - first) / units + 1) : 0;
    last_n = kSub && left && first + (left - 1) * units == t.units - 1 ? static_cast<int>(static_cast<uint32_t>(a.rows) - (t.units - 1) * rows) : rows;
    base = smem + me.team * t.stages * MATS * t.mat_bytes;
    bars = smem_u32(smem + t.off_bar) + 8 * me.team * t.stages;
    abort_flag = reinterpret_cast<volatile int*>(smem + t.off_bar + 8 * t.stages * me.teams);
    stage = 0, phase = 0;
    if (me.warp == 0 && (threadIdx.x & 31) == 0)
      for (int i = 0; i < t.stages; ++i) mbar_init(bars + 8 * i, 1);
    if (threadIdx.x == 0) *abort_flag = 0;
    if ((threadIdx.x & 31) == 0) mbar_fence_init();
    __syncthreads();
  }
  // called by the team's first warp: the unit `ahead` behind the present one
  __device__ __forceinline__ void load(int ahead, int st) {
    if (ahead >= left) return;
    const T* src[MATS];
    long long ld[MATS];
    src[0] = static_cast<const T*>(a.x), ld[0] = a.ldx;
    if constexpr (MATS == 2) src[1] = static_cast<const T*>(a.dy), ld[1] = a.lddy;
    load_stage<T, VEC, MATS>(src, ld, a, t, row + ahead * step, ahead == left - 1 ? last_n : kSub ? t.rows : 1, base + st * MATS * t.mat_bytes, bars + 8 * st);
  }
  __device__ __forceinline__ void fill() {
    for (int i = 0; i < t.stages; ++i) load(i, i);
  }
  __device__ __forceinline__ bool wait(int site) { return mbar_wait_warp(bars + 8 * stage, phase, abort_flag, t.dev_status, site); }
  __device__ __forceinline__ const T* mat(int m) const {
    return reinterpret_cast<const T*>(base + (stage * MATS + m) * t.mat_bytes) + stage_shift<T, VEC>(row, a.C);
  }
  // whether row `sub` of the unit `ahead` behind the present one exists
  __device__ __forceinline__ bool has(int ahead, int sub) const { return ahead < left - 1 || (ahead == left - 1 && sub < last_n); }
  // after the team has read the stage: called by its first warp
  __device__ __forceinline__ void refill() { load(t.stages, stage); }
  __device__ __forceinline__ void next_stage() {
    if (++stage == t.stages) stage = 0, phase ^= 1u;
  }
  __device__ __forceinline__ void next_unit() { row += step, --left; }
};

// Rows of 16-bit values take up to eight vectors a thread, so that few warps share a row (sums across warps, waits and refills are
// most of the other instructions); beyond three, weight and bias do not fit in registers beside them and are read from shared
// memory.  64M values of fp16, at most three vectors / up to eight: 1280 columns 51.7 / 45.1 us, 1608 75 / 46.0, 4096 62 / 46.1.  (Rows
// of single values: beyond 16 of them.)
template <int VEC, int NV>
__host__ __device__ constexpr bool fwd_params_shared() { return VEC == 1 ? NV > 16 : VEC == 8 && NV > 3; }
// Bound by memory: 65536 x 1280 fp16 58 us (5.8 TB/s, 89 % of a copy's rate; 61 on a slower GPU), 50000 x 1280 fp32 90 us (5.7 TB/s).
template <class T, int VEC, int NV, int kTeams>
__global__ void __launch_bounds__(kTeamThreads, NV * VEC <= 8 ? 2 : 1) ln_fwd_teams_kernel(const LnArgs a, const LnTeams t) {
  constexpr bool kSub = kTeams != kWide;
  pdl_launch_dependents();
  using F = typename Lanes<VEC>::F;
  constexpr int N = Lanes<VEC>::N;
  extern __shared__ __align__(128) uint8_t smem[];
  const TeamRole me(t.TL);
  TeamRing<T, VEC, 1, kSub> ring(a, t, smem, me);
  float* slots = reinterpret_cast<float*>(smem + t.off_red);
  const int n = a.C / VEC;
  pdl_wait();
  if (me.warp == 0) ring.fill();
  constexpr bool kShared = fwd_params_shared<VEC, NV>();
  float* sw = reinterpret_cast<float*>(smem + t.off_w);
  F w[kShared ? 1 : NV][N], b[kShared ? 1 : NV][N];
  {
    const Param<T> pw{a.weight, a.param_f32}, pb{a.bias, a.param_f32};
    if constexpr (kShared) {
      for (int c = threadIdx.x; c < a.C; c += kTeamThreads) {
        const int at = shared_param_index<VEC>(n, c);
        sw[at] = pw.p ? pw.at(c) : 1.f, sw[a.C + at] = pb.p ? pb.at(c) : 0.f;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = min(me.lane + i * t.TL, n - 1);
        pw.template get<VEC>((long long)v * VEC, 1.f, w[i]);
        pb.template get<VEC>((long long)v * VEC, 0.f, b[i]);
      }
    }
  }
  bool failed = false;
  const int groups = kTeams == kGrouped ? t.groups : 1;
  for (; ring.left > 0 && !failed; ring.next_unit()) {
    failed = !ring.wait(700);
    if (kSub && failed) break;
    const T* xs = ring.mat(0) + (kSub ? me.sub * a.C : 0);
    for (int sub = kSub ? me.sub : 0, g = 1; g <= groups; ++g, sub += t.per, xs += t.per * a.C) {
      const uint32_t row = ring.row + sub;
      const bool in = !kSub || ring.has(0, sub);
      F x[NV][N];
      F s[2] = {splat<F>(0.f), splat<F>(0.f)};   // two chains of additions
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = me.lane + i * t.TL;
        if (in && has_vector<VEC, NV>(i, v, n)) {
          widen<T, VEC>(load_vec<T, VEC>(xs + v * VEC), x[i]);
#pragma unroll
          for (int j = 0; j < N; ++j) s[(i * N + j) % 2] = add(s[(i * N + j) % 2], x[i][j]);
        }
      }
      float sum[1] = {total(add(s[0], s[1]))};
      failed = team_sum<1, kSub>(sum, t, me, slots, 0, failed);
      if (failed) break;
      if (g == groups) {   // the stage has been read by the whole team
        __syncwarp();
        if (me.warp == 0) ring.refill();
        ring.next_stage();
      }
      const float mean = mean_of(sum[0], a);
      const F minus = splat<F>(-mean);
      s[0] = s[1] = splat<F>(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (has_vector<VEC, NV>(i, me.lane + i * t.TL, n)) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            x[i][j] = add(x[i][j], minus);
            s[(i * N + j) % 2] = fma(x[i][j], x[i][j], s[(i * N + j) % 2]);
          }
        }
      }
      sum[0] = total(add(s[0], s[1]));
      team_sum<1, kSub>(sum, t, me, slots, 1, false);
      const float rstd = rsqrtf(sum[0] * a.inv_c + a.eps);
      if (in) {
        const F scale = splat<F>(rstd);
        T* yr = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = me.lane + i * t.TL;
          if (has_vector<VEC, NV>(i, v, n)) {
            if constexpr (kShared) shared_param<VEC>(sw, n, v, w[0]), shared_param<VEC>(sw + a.C, n, v, b[0]);
            constexpr int k = kShared ? 0 : 1;
#pragma unroll
            for (int j = 0; j < N; ++j) x[i][j] = fma(mul(x[i][j], scale), w[k * i][j], b[k * i][j]);
            store_vec<T, VEC>(yr + v * VEC, narrow<T, VEC>(x[i]));
          }
        }
        if (a.mean && me.lane == 0) a.mean[row] = mean, a.rstd[row] = rstd;
      }
    }
  }
  if (__syncthreads_or(failed)) let_copies_land();
}

// ---- backward --------------------------------------------------------------------------------
// fp32 rows are bound by memory (8192 x 5120 76 us without the column sums' second launch, 6.6 TB/s), 16-bit ones by the 16 warps an SM that
// the sums' registers allow (58 to 60 % of the issue slots taken): 50000 x 1280 71 us, 5.4 TB/s; 32768 x 640 27 us and 4.7 for
// the second launch.
template <class T, int VEC, int NV, int kTeams>
__global__ void __launch_bounds__(kTeamThreads, 1) ln_bwd_teams_kernel(const LnArgs a, const LnTeams t) {
  constexpr bool kSub = kTeams != kWide;
  pdl_launch_dependents();
  using F = typename Lanes<VEC>::F;
  constexpr int N = Lanes<VEC>::N;
  extern __shared__ __align__(128) uint8_t smem[];
  const TeamRole me(t.TL);
  TeamRing<T, VEC, 2, kSub> ring(a, t, smem, me);
  float* slots = reinterpret_cast<float*>(smem + t.off_red);
  float* sw = reinterpret_cast<float*>(smem + t.off_w);
  const int n = a.C / VEC;
  pdl_wait();
  if (me.warp == 0) ring.fill();
  {
    const Param<T> w{a.weight, a.param_f32};
    for (int c = threadIdx.x; c < a.C; c += kTeamThreads) sw[shared_param_index<VEC>(n, c)] = w.p ? w.at(c) : 1.f;
  }
  F dw[NV][N], db[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) dw[i][j] = db[i][j] = splat<F>(0.f);
  float mean_next = 0.f, rstd_next = 0.f;
  auto moments = [&](int ahead, int sub) {
    const uint32_t r = ring.row + ahead * ring.step + sub;
    if (ring.has(ahead, sub)) mean_next = a.mean[r], rstd_next = a.rstd[r];
  };
  moments(0, me.sub);
  __syncthreads();
  bool failed = false;
  const int groups = kTeams == kGrouped ? t.groups : 1;
  for (; ring.left > 0 && !failed; ring.next_unit()) {
    failed = !ring.wait(701);
    if (kSub && failed) break;
    const T* xs = ring.mat(0) + (kSub ? me.sub * a.C : 0);
    const T* ds = ring.mat(1) + (kSub ? me.sub * a.C : 0);
    for (int sub = kSub ? me.sub : 0, g = 1; g <= groups; ++g, sub += t.per, xs += t.per * a.C, ds += t.per * a.C) {
      const bool in = !kSub || ring.has(0, sub);
      Vec<T, VEC> rx[NV], rd[NV];          // as loaded, and widened twice: registers bound this kernel
      const float mean = mean_next, rstd = rstd_next;
      if (g < groups) moments(0, sub + t.per);
      else moments(1, kSub ? me.sub : 0);
      F s1 = splat<F>(0.f), s2 = s1;       // sum(g), sum(g (x - mean))
      const F minus = splat<F>(-mean);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = me.lane + i * t.TL;
        if (in && has_vector<VEC, NV>(i, v, n)) {
          F w[N], d[N], x[N];
          rx[i] = load_vec<T, VEC>(xs + v * VEC), rd[i] = load_vec<T, VEC>(ds + v * VEC);
          widen<T, VEC>(rx[i], x), widen<T, VEC>(rd[i], d);
          shared_param<VEC>(sw, n, v, w);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const F g = mul(d[j], w[j]);
            s1 = add(s1, g);
            s2 = fma(g, add(x[j], minus), s2);
          }
        }
      }
      float sum[2] = {total(s1), total(s2)};
      failed = team_sum<2, kSub>(sum, t, me, slots, ring.left & 1, failed);
      if (failed) break;
      if (g == groups) {   // the stage has been read by the whole team
        __syncwarp();
        if (me.warp == 0) ring.refill();
        ring.next_stage();
      }
      const F r = splat<F>(rstd), c1 = splat<F>(-rstd * (sum[0] * a.inv_c)), c2 = splat<F>(-rstd * (rstd * (sum[1] * a.inv_c)));
      if (in) {
        T* out = static_cast<T*>(a.y) + (ring.row + sub) * a.ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = me.lane + i * t.TL;
          if (has_vector<VEC, NV>(i, v, n)) {
            F w[N], d[N], x[N];
            widen<T, VEC>(rx[i], x), widen<T, VEC>(rd[i], d);
            shared_param<VEC>(sw, n, v, w);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              // dx = dy (w r) + h c2 + c1
              const F h = mul(add(x[j], minus), r);
              dw[i][j] = fma(d[j], h, dw[i][j]);
              db[i][j] = add(db[i][j], d[j]);
              x[j] = fma(d[j], mul(w[j], r), fma(h, c2, c1));
            }
            store_vec<T, VEC>(out + v * VEC, narrow<T, VEC>(x));
          }
        }
      }
    }
  }
  if (__syncthreads_or(failed)) {
    let_copies_land();
    return;
  }
  if (!a.part) return;
  // Column sums of the block: over the rows of a warp by shuffles, over teams through shared memory (the rings are empty by
  // now).
  if constexpr (kSub) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j)
        for (int o = t.TL; o < 32; o <<= 1) {
          if constexpr (VEC == 1) {
            dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], o), db[i][j] += __shfl_xor_sync(0xffffffffu, db[i][j], o);
          } else {
            dw[i][j] = add(dw[i][j], F2{__shfl_xor_sync(0xffffffffu, dw[i][j].v, o)});
            db[i][j] = add(db[i][j], F2{__shfl_xor_sync(0xffffffffu, db[i][j].v, o)});
          }
        }
  }
  float* sums = a.part + blockIdx.x * 2ll * a.C;
  float* to = me.teams > 1 ? reinterpret_cast<float*>(smem) + me.team * 2 * a.C : sums;
  if (me.sub == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = me.lane + i * t.TL;
      if (has_vector<VEC, NV>(i, v, n)) {
        *reinterpret_cast<Vec<F, N>*>(to + v * VEC) = *reinterpret_cast<const Vec<F, N>*>(&dw[i]);
        *reinterpret_cast<Vec<F, N>*>(to + a.C + v * VEC) = *reinterpret_cast<const Vec<F, N>*>(&db[i]);
      }
    }
  }
  if (me.teams == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.C; c += kTeamThreads) {
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < me.teams; ++k) s += reinterpret_cast<const float*>(smem)[k * 2 * a.C + c];
    sums[c] = s;
  }
}

// Few rows, in one launch: the first `a.rows` blocks form a row of dx each, the others 32 columns of dw and db each.  Both read x
// and dy, which by then lie in L2; no partial sums, no second launch (154 x 2048: 7.5 -> 2.8 us; 512 x 1280: 8.0 -> 7.4, 1024 x
// 1280: 8.7 against 14.2).
constexpr int kSmallThreads = 512, kSmallRows = 512;
template <class T, class P, int VEC>
__global__ void __launch_bounds__(kSmallThreads) ln_bwd_small_kernel(const LnArgs a, P* dweight, P* dbias) {
  pdl_launch_dependents();
  using F = typename Lanes<VEC>::F;
  constexpr int N = Lanes<VEC>::N, kWarps = kSmallThreads / 32;
  __shared__ float red[2][kWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  if (blockIdx.x < a.rows) {
    const long long r = blockIdx.x;
    const Param<T> w{a.weight, a.param_f32};
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dr = static_cast<const T*>(a.dy) + r * a.lddy;
    const float mean = a.mean[r], rstd = a.rstd[r];
    const F minus = splat<F>(-mean);
    const int n = a.C / VEC;
    F s1 = splat<F>(0.f), s2 = s1;
    for (int v = threadIdx.x; v < n; v += kSmallThreads) {
      F x[N], d[N], wv[N];
      widen<T, VEC>(load_vec<T, VEC>(xr + v * VEC), x), widen<T, VEC>(load_vec<T, VEC>(dr + v * VEC), d);
      w.template get<VEC>(v * VEC, 1.f, wv);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const F g = mul(d[j], wv[j]);
        s1 = add(s1, g);
        s2 = fma(g, add(x[j], minus), s2);
      }
    }
    const float t1 = block_sum(total(s1), red[0][0]) * a.inv_c, t2 = block_sum(total(s2), red[1][0]) * a.inv_c;
    const F rs = splat<F>(rstd), c1 = splat<F>(-rstd * t1), c2 = splat<F>(-rstd * (rstd * t2));
    T* out = static_cast<T*>(a.y) + r * a.ldy;
    for (int v = threadIdx.x; v < n; v += kSmallThreads) {
      F x[N], d[N], wv[N];
      widen<T, VEC>(load_vec<T, VEC>(xr + v * VEC), x), widen<T, VEC>(load_vec<T, VEC>(dr + v * VEC), d);
      w.template get<VEC>(v * VEC, 1.f, wv);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = fma(d[j], mul(wv[j], rs), fma(mul(add(x[j], minus), rs), c2, c1));
      store_vec<T, VEC>(out + v * VEC, narrow<T, VEC>(x));
    }
    return;
  }
  const int c = (blockIdx.x - static_cast<int>(a.rows)) * 32 + lane;
  float dw = 0.f, db = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int r = warp; r < a.rows; r += kWarps) {
      const float d = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
      dw = fmaf(d, (to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r], dw);
      db += d;
    }
  }
  red[0][warp][lane] = dw, red[1][warp][lane] = db;
  __syncthreads();
  P* out = warp == 0 ? dweight : dbias;
  if (warp > 1 || c >= a.C || !out) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) v += red[warp][k][lane];
  out[c] = from_f32<P>(v);
}

// Rows that the teams do not take: dx alone, two passes over the row.
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
#pragma unroll 8
    for (int i = warp; i < count; i += warps) v += part[i * pitch + blockIdx.y * (long long)C + c];
  s[warp][lane] = v;
  __syncthreads();
  for (int k = warp; k < 32; k += warps) {
    float sum[1] = {lane < warps ? s[lane][k] : 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) add_lanes<1>(sum, o);
    if (lane == 0 && blockIdx.x * 32 + k < C) out[blockIdx.x * 32 + k] = from_f32<P>(sum[0]);
  }
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

// Once per kernel and device: more dynamic shared memory than the default.
template <auto kernel>
static int allow_smem(int bytes) {
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute(layernorm)")) return rc;
    configured[dev] = true;
  }
  return kOk;
}
constexpr int kLnMaxC = 1 << 30;   // column indices, and a step past the last one, are ints
// Rows of column sums that the backward pass leaves, at most: one per block of the teams (one an SM), or per share of ln_bwd_columns_kernel.
constexpr int kColumnShares = 64;
static long long ln_bwd_blocks(long long rows) {
  if (rows <= kSmallRows) return 0;
  const long long most = sm_count() > kColumnShares ? sm_count() : kColumnShares;
  return rows < most ? rows : most;
}

// Whether rows of `base` lie back to back from a 16-byte aligned address on.
static bool back_to_back(const void* base, long long ld, int C) { return al16(base) && ld == C; }

constexpr long long kSmemSm = 227 * 1024, kSmemHalf = kSmemSm / 2 - 1024;   // of an SM; a block's where two share one
// Fills `t` for rows of `mats` matrices and threads of at most `most` vectors (`most_sub` in teams of up to a warp); false where rows of this size do not fit.
// `grouped`: up to how many vectors a thread there are kernels that take several rows of a team as one unit (others would leave out all
// but the first).  `params`: bytes of shared memory for the parameters; `sums`: whether the block's column sums meet in the rings at the end;
// `room`: shared memory of a block.  NV of the kernel: t.nv.
static bool plan_teams(LnTeams& t, const LnArgs& a, int elem, int vec, int mats, int most_sub, int most, int grouped, long long params, bool sums, long long room, int& nv,
                       int& smem) {
  const long long row = a.C * (long long)elem, n = a.C / vec;
  if (a.rows > INT_MAX) return false;
  int TL = 8;
  while (TL < kTeamThreads && n > (TL > 32 ? most : most_sub) * (long long)TL) TL *= 2;
  if (n > (long long)most * TL) return false;
  nv = (int)((n + TL - 1) / TL);
  if (vec == 1) nv = (nv + 3) / 4 * 4;
  const int warps = TL > 32 ? TL / 32 : 1, teams = kTeamWarps / warps;
  t.ceiling = (unsigned long long)a.rows * a.C / (16 / elem) * (16 / elem);
  const long long slots = 2ll * kTeamWarps * mats * 4, rest = params + slots + teams * 8 * 8 + 512;
  const long long scratch = sums && teams > 1 ? teams * 2ll * a.C * 4 : 0;
  auto bytes = [&](long long rows) { return (rows * row + 15) / 16 * 16 + (vec == 1 ? 32 : 0); };   // a widened span begins and ends up to 15 bytes further out
  auto stages_of = [&](long long rows) { return (room - rest) / (teams * mats * bytes(rows)); };
  // A warp's waits and refills cost as many instructions as 600 values of a row: several rows of 16-bit values share them, as long as two
  // stages remain (three forward: with two, 100000 x 640 49.1 us for 43.8) and every team has six units or more.  fp16 backward of 1000000 x
  // 64 93.5 -> 80.7 us, 100000 x 640 80.0 -> 77.6; fp32 and rows that are not 16-byte aligned gain nothing (65536 x 320 fp32 29.7, 32.3).
  t.TL = TL, t.per = TL < 32 ? 32 / TL : 1, t.groups = 1;
  const long long grid_teams = (long long)teams * sm_count() * (room < kSmemSm ? 2 : 1);
  while (elem == 2 && vec > 1 && TL <= 32 && nv <= grouped && t.groups < 8 && stages_of(2ll * t.groups * t.per) >= (mats == 1 ? 3 : 2) &&
         a.rows >= 6 * grid_teams * 2 * t.groups * t.per)
    t.groups *= 2;
  t.rows = t.per * t.groups, t.units = (uint32_t)((a.rows + t.rows - 1) / t.rows);
  t.mat_bytes = (int)bytes(t.rows);
  long long stages = stages_of(t.rows);
  if (stages > 8) stages = 8;
  if (stages < 2 || scratch > room - rest) return false;
  t.stages = (int)stages;
  long long ring = stages * teams * mats * t.mat_bytes;
  if (ring < scratch) ring = scratch;
  t.off_w = (int)((ring + 127) / 128 * 128);
  t.off_red = (int)((t.off_w + params + 15) / 16 * 16);
  t.off_bar = (int)(t.off_red + slots);
  smem = t.off_bar + 8 * t.stages * teams + 16;
  return smem <= room;
}
static int team_blocks(const LnTeams& t, int per_sm) {
  const long long teams = kTeamWarps / (t.TL > 32 ? t.TL / 32 : 1), need = ((long long)t.units + teams - 1) / teams, most = (long long)sm_count() * per_sm;
  return (int)(need < most ? need : most);
}

// Vectors a thread holds in teams of up to a warp (eight of 16-bit values spill there: 2048 columns 52.4 us, with seven 46.6).
template <int VEC>
constexpr int fwd_most_sub() { return VEC == 1 ? 24 : VEC == 8 ? 7 : 6; }
constexpr int kFwdGrouped = 5;   // (three stages of two wider rows each do not fit)
template <class T, int VEC, int NV, int kTeams = kWide>
static int ln_fwd_teams_launch(const LnArgs& a, const LnTeams& t, int smem, cudaStream_t s) {
  if constexpr (kTeams == kWide && NV <= fwd_most_sub<VEC>()) {
    if constexpr (sizeof(T) == 2 && VEC > 1 && NV <= kFwdGrouped)
      if (t.groups > 1) return ln_fwd_teams_launch<T, VEC, NV, kGrouped>(a, t, smem, s);
    if (t.TL <= 32) return ln_fwd_teams_launch<T, VEC, NV, kNarrow>(a, t, smem, s);
  }
  if constexpr (kTeams == kWide && 2 * NV <= (VEC == 1 ? 12 : fwd_most_sub<VEC>())) {
    return fail(kErrUnsupported, "bxl_layernorm_fwd: no team of several warps has rows this narrow");
  } else {
    if (int rc = allow_smem<ln_fwd_teams_kernel<T, VEC, NV, kTeams>>(kSmemSm)) return rc;
    return launch_kernel("ln_fwd_teams_kernel launch", ln_fwd_teams_kernel<T, VEC, NV, kTeams>, dim3(team_blocks(t, smem <= kSmemHalf ? 2 : 1)), dim3(kTeamThreads), smem, s, 1, a, t);
  }
}
template <class T, int VEC>
static int ln_fwd_teams(const LnArgs& a, bool& done, cudaStream_t s) {
  LnTeams t = {};
  int nv = 0, smem = 0;
  const bool close = back_to_back(a.x, a.ldx, a.C);
  constexpr int sub = fwd_most_sub<VEC>(), most = VEC == 8 ? 8 : sub, wide = 8;
  const long long params = VEC == 4 ? 0 : 8ll * a.C;
  // Single values: up to 24 a thread where every team has eight units or more, else 12 for more teams (100000 x 643 fp16 104 us with 12,
  // 88 with 24; 4099 x 1285 fp32 12.4 and 13.8), or what the widest rows need (5000 x 12001: without a ring 234 us, 88 so).
  auto plan = [&](int narrow, int wider, long long room) { return plan_teams(t, a, sizeof(T), VEC, 1, narrow, wider, kFwdGrouped, params, false, room, nv, smem); };
  int narrow = sub, wider = most;
  done = (VEC > 1 || close) && plan(narrow, wider, kSmemSm);
  if (VEC == 1 && done && t.units < 8ll * sm_count() * (t.TL > 32 ? kTeamThreads / t.TL : kTeamWarps)) {
    narrow = wider = 12;
    if (!plan(narrow, wider, kSmemSm)) narrow = wider = sub, plan(narrow, wider, kSmemSm);
  }
  if (VEC == 4 && !done) wider = wide, done = plan(narrow, wider, kSmemSm);
  if (done && nv * VEC <= 8 && !plan(narrow, wider, kSmemHalf)) plan(narrow, wider, kSmemSm);   // two blocks an SM
  if (!done) return kOk;
  t.one_copy = close || t.rows == 1;
  if (!(t.dev_status = device_status_ptr())) return fail(kErrCuda, "bxl_layernorm_fwd: no device status word");
  if constexpr (VEC == 1) {
    if (nv <= 4) return ln_fwd_teams_launch<T, 1, 4>(a, t, smem, s);
    if (nv <= 8) return ln_fwd_teams_launch<T, 1, 8>(a, t, smem, s);
    if (nv <= 12) return ln_fwd_teams_launch<T, 1, 12>(a, t, smem, s);
    if (nv <= 16) return ln_fwd_teams_launch<T, 1, 16>(a, t, smem, s);
    if (nv <= 20) return ln_fwd_teams_launch<T, 1, 20>(a, t, smem, s);
    return ln_fwd_teams_launch<T, 1, 24>(a, t, smem, s);
  } else {
    if (nv == 1) return ln_fwd_teams_launch<T, VEC, 1>(a, t, smem, s);
    if (nv == 2) return ln_fwd_teams_launch<T, VEC, 2>(a, t, smem, s);
    if (nv == 3) return ln_fwd_teams_launch<T, VEC, 3>(a, t, smem, s);
    if (nv == 4) return ln_fwd_teams_launch<T, VEC, 4>(a, t, smem, s);
    if (nv == 5) return ln_fwd_teams_launch<T, VEC, 5>(a, t, smem, s);
    if (nv == 6) return ln_fwd_teams_launch<T, VEC, 6>(a, t, smem, s);
    if (nv == 7) return ln_fwd_teams_launch<T, VEC, 7>(a, t, smem, s);
    return ln_fwd_teams_launch<T, VEC, 8>(a, t, smem, s);
  }
}

template <class T, int VEC, int NV, int LANES, int kMaxThreads = LANES ? kLnWarps * 32 : 512>
static int ln_fwd_launch(const LnArgs& a, int threads, cudaStream_t s) {
  constexpr int kRows = LANES ? kLnWarps * 32 / LANES : 1;
  const long long need = (a.rows + kRows - 1) / kRows, most = sm_count() * (2048ll / threads);
  return launch_kernel("ln_fwd_kernel launch", ln_fwd_kernel<T, VEC, NV, LANES, kMaxThreads>, dim3((unsigned)(need < most ? need : most)), dim3(threads), 0, s, 1, a);
}
template <class T>
static int ln_fwd(const LnArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T), W = kLnWarps * 32;
  // Few values: a block's ring costs more than it brings (1024 x 640: 3.0 us without, 3.4 with; 4096 x 320: 4.3 and 3.8).
  const long long few = vec ? 1 << 20 : 1 << 18;
  if (a.rows * a.C > few) {
    bool done = false;
    if (int rc = vec ? ln_fwd_teams<T, V>(a, done, s) : ln_fwd_teams<T, 1>(a, done, s)) return rc;
    if (done) return kOk;
  }
  if (vec) {
    const int n = a.C / V;
    if (n <= 32) return ln_fwd_launch<T, V, 1, 32>(a, W, s);
    if (n <= 64) return ln_fwd_launch<T, V, 2, 32>(a, W, s);
    if (n <= 96) return ln_fwd_launch<T, V, 3, 32>(a, W, s);
    for (int threads = 64; threads <= 512; threads *= 2)
      if (n <= 2 * threads) return ln_fwd_launch<T, V, 2, 0>(a, threads, s);
    if (n <= 2048) return ln_fwd_launch<T, V, 4, 0>(a, 512, s);
    if (n <= 4096) return ln_fwd_launch<T, V, 4, 0, 1024>(a, 1024, s);
  } else {
    if (a.C <= 256) return ln_fwd_launch<T, 1, 8, 32>(a, W, s);
    if (a.C <= 2048) return ln_fwd_launch<T, 1, 8, 0>(a, 256, s);
    if (a.C <= 8192) return ln_fwd_launch<T, 1, 8, 0, 1024>(a, 1024, s);
  }
  const long long most = (long long)sm_count() * 2;
  return launch_kernel("ln_fwd_long_kernel launch", ln_fwd_long_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(1024), 0, s, 1, a);
}

// Vectors a thread holds: 24 values of 16 bits or 16 of fp32 (8192 x 5120: 96 us with 24, 86 with 16); wider rows spill.  Single values: 16 of
// 16 bits (38611 x 1819 fp16 165 us with 12, 125 with 16), 12 of fp32; 24 in rows that are wider than that, spilling (5000 x 12001 fp16
// 330 us without a ring, 180 so).
template <class T, int VEC>
constexpr int bwd_most() { return VEC == 1 ? (sizeof(T) == 2 ? 16 : 12) : VEC == 8 ? 3 : 4; }
template <class T, int VEC, int NV, int kTeams = kWide>
static int ln_bwd_teams_launch(const LnArgs& a, const LnTeams& t, int blocks, int smem, cudaStream_t s) {
  if constexpr (kTeams == kWide && NV <= (VEC == 4 && sizeof(T) == 2 ? 5 : bwd_most<T, VEC>())) {
    if constexpr (sizeof(T) == 2 && VEC > 1)
      if (t.groups > 1) return ln_bwd_teams_launch<T, VEC, NV, kGrouped>(a, t, blocks, smem, s);
    if (t.TL <= 32) return ln_bwd_teams_launch<T, VEC, NV, kNarrow>(a, t, blocks, smem, s);
  }
  if constexpr (kTeams == kWide && 2 * NV <= (VEC == 4 && sizeof(T) == 2 ? 6 : bwd_most<T, VEC>())) {
    return fail(kErrUnsupported, "bxl_layernorm_bwd: no team of several warps has rows this narrow");
  } else {
    if (int rc = allow_smem<ln_bwd_teams_kernel<T, VEC, NV, kTeams>>(kSmemSm)) return rc;
    return launch_kernel("ln_bwd_teams_kernel launch", ln_bwd_teams_kernel<T, VEC, NV, kTeams>, dim3(blocks), dim3(kTeamThreads), smem, s, 1, a, t);
  }
}
template <class T, int VEC>
static int ln_bwd_teams(const LnArgs& a, bool& done, int& blocks, cudaStream_t s) {
  LnTeams t = {};
  int nv = 0, smem = 0;
  const bool close = back_to_back(a.x, a.ldx, a.C) && back_to_back(a.dy, a.lddy, a.C);
  constexpr int most = bwd_most<T, VEC>(), wide = VEC == 1 ? 24 : VEC == 8 ? 4 : 6;
  done = (VEC > 1 || close) && (plan_teams(t, a, sizeof(T), VEC, 2, most, most, most, 4ll * a.C, true, kSmemSm, nv, smem) ||
                                         plan_teams(t, a, sizeof(T), VEC, 2, most, wide, most, 4ll * a.C, true, kSmemSm, nv, smem));
  if (!done) return kOk;
  t.one_copy = close || t.rows == 1;
  if (!(t.dev_status = device_status_ptr())) return fail(kErrCuda, "bxl_layernorm_bwd: no device status word");
  blocks = team_blocks(t, 1);
  if constexpr (VEC == 1) {
    if (nv <= 4) return ln_bwd_teams_launch<T, 1, 4>(a, t, blocks, smem, s);
    if (nv <= 8) return ln_bwd_teams_launch<T, 1, 8>(a, t, blocks, smem, s);
    if (nv <= 12) return ln_bwd_teams_launch<T, 1, 12>(a, t, blocks, smem, s);
    if (nv <= 16) return ln_bwd_teams_launch<T, 1, 16>(a, t, blocks, smem, s);
    if (nv <= 20) return ln_bwd_teams_launch<T, 1, 20>(a, t, blocks, smem, s);
    return ln_bwd_teams_launch<T, 1, 24>(a, t, blocks, smem, s);
  } else {
    // Vectors of 8 bytes where those of 16 would leave a sixth or more of the last ones' lanes idle (64M values of fp16: 640 columns 87.6 us
    // with 16 bytes, 82.0 with 8; 1280 78.4 and 72.1; 3436 x 13440, where both spill, 106 and 95).
    if constexpr (VEC == 8) {
      const int half = (a.C / 4 + t.TL - 1) / t.TL;
      if (half == 3) return ln_bwd_teams_launch<T, 4, 3>(a, t, blocks, smem, s);
      if (half == 5) return ln_bwd_teams_launch<T, 4, 5>(a, t, blocks, smem, s);
      if (half == 7) return ln_bwd_teams_launch<T, 4, 7>(a, t, blocks, smem, s);
    }
    if (nv == 1) return ln_bwd_teams_launch<T, VEC, 1>(a, t, blocks, smem, s);
    if (nv == 2) return ln_bwd_teams_launch<T, VEC, 2>(a, t, blocks, smem, s);
    if (nv == 3) return ln_bwd_teams_launch<T, VEC, 3>(a, t, blocks, smem, s);
    if (nv == 4) return ln_bwd_teams_launch<T, VEC, 4>(a, t, blocks, smem, s);
    if constexpr (VEC == 4) {
      if (nv == 5) return ln_bwd_teams_launch<T, VEC, 5>(a, t, blocks, smem, s);
      return ln_bwd_teams_launch<T, VEC, 6>(a, t, blocks, smem, s);
    }
    return fail(kErrUnsupported, "bxl_layernorm_bwd: no kernel for %d vectors a thread", nv);
  }
}

template <class T, class P>
static int ln_bwd_small(const LnArgs& a, bool vec, void* dweight, void* dbias, cudaStream_t s) {
  const dim3 grid((unsigned)a.rows + (dweight || dbias ? (a.C + 31) / 32 : 0));
  constexpr int V = 16 / sizeof(T);
  P *dw = static_cast<P*>(dweight), *db = static_cast<P*>(dbias);
  if (vec) return launch_kernel("ln_bwd_small_kernel launch", ln_bwd_small_kernel<T, P, V>, grid, dim3(kSmallThreads), 0, s, 1, a, dw, db);
  return launch_kernel("ln_bwd_small_kernel launch", ln_bwd_small_kernel<T, P, 1>, grid, dim3(kSmallThreads), 0, s, 1, a, dw, db);
}
static thread_local int g_bwd_launches = 0;
template <class T>
static int ln_bwd(const LnArgs& a, bool vec, int& blocks, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  bool done = false;
  if (int rc = vec ? ln_bwd_teams<T, V>(a, done, blocks, s) : ln_bwd_teams<T, 1>(a, done, blocks, s)) return rc;
  if (done) return kOk;
  const long long most = (long long)sm_count() * 2;
  if (int rc = launch_kernel("ln_bwd_long_kernel launch", ln_bwd_long_kernel<T>, dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(1024), 0, s, 1, a))
    return rc;
  if (!a.part) return kOk;
  const long long shares = a.rows < kColumnShares ? a.rows : kColumnShares;
  blocks = (int)shares;
  ++g_bwd_launches;
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
  const long long bytes = ln_bwd_blocks(rows) * 2ll * C * (long long)sizeof(float);
  return bytes ? bytes + kPartSlack : 0;
}

extern "C" int bxl_layernorm_bwd_launches(void) { return g_bwd_launches; }

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
  if (params && ln_bwd_blocks(rows)) {
    if (!workspace || !al16(workspace)) return fail(kErrInvalidArg, "bxl_layernorm_bwd: workspace must be 16-byte aligned");
    if (workspace_bytes < bxl_layernorm_bwd_workspace_bytes(rows, C)) return fail(kErrTooLarge, "bxl_layernorm_bwd: workspace too small");
  }
  LnArgs a = {};
  a.x = x, a.dy = dy, a.y = dx, a.ldx = ldx, a.lddy = lddy, a.ldy = lddx, a.weight = weight;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.part = params ? part_base(workspace) : nullptr;
  a.rows = rows, a.C = C, a.param_f32 = param_dtype == BXL_F32, a.inv_c = 1.f / (float)C;
  const bool vec = rows_of_vectors(x, ldx, C, b) && rows_of_vectors(dy, lddy, C, b) && rows_of_vectors(dx, lddx, C, b) && al16(weight);
  cudaStream_t s = (cudaStream_t)stream;
  g_bwd_launches = 1;
  if (!ln_bwd_blocks(rows)) {
    a.part = nullptr;
    if (dtype == BXL_F32) return ln_bwd_small<float, float>(a, vec, dweight, dbias, s);
    if (dtype == BXL_F16) return param_dtype == BXL_F32 ? ln_bwd_small<__half, float>(a, vec, dweight, dbias, s) : ln_bwd_small<__half, __half>(a, vec, dweight, dbias, s);
    return param_dtype == BXL_F32 ? ln_bwd_small<__nv_bfloat16, float>(a, vec, dweight, dbias, s) : ln_bwd_small<__nv_bfloat16, __nv_bfloat16>(a, vec, dweight, dbias, s);
  }
  int blocks = 0, rc;
  if (dtype == BXL_F16) rc = ln_bwd<__half>(a, vec, blocks, s);
  else if (dtype == BXL_BF16) rc = ln_bwd<__nv_bfloat16>(a, vec, blocks, s);
  else rc = ln_bwd<float>(a, vec, blocks, s);
  if (rc || !params) return rc;
  ++g_bwd_launches;
  return sum_partials(a.part, blocks, 2ll * C, C, dweight, dbias, param_dtype, s);
}
