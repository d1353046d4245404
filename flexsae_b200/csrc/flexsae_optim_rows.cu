// AdamW on a decoder whose rows are kept at unit length: projection of the gradient, step and division by the
// row's length in one pass.
//
// A team of threads holds a row, eight elements each, so it stays in registers between its three uses: the CTA, or,
// for rows of up to 256 elements, a warp or a power-of-two part of one (no barrier then).  A row is read and written
// once; 65536 rows of 2304 bf16 take 0.52 ms, 98 % of the HBM rate.
#include <type_traits>

#include "flexsae_optim.cuh"

namespace flexsae {

// Where the eight elements of a thread lie.
enum RowMode {
  kWholeRows,      // aligned tensors whose rows are whole groups of eight: a group per thread
  kGroupedRows,    // aligned tensors, rows of any length: the groups of eight that a row touches, the first and the last
                   // of which may belong to it in part
  kStridedRows,    // every team-th element
};

// The thread's elements of the row of `n` elements (0: no row) that starts at `begin`; zero where it has none.
template <RowMode MODE, typename T>
__device__ __forceinline__ void row_load(const void* base, long long begin, int n, int lane, int team, float2* out) {
  const T* q = reinterpret_cast<const T*>(base);
  float* f = reinterpret_cast<float*>(out);
  if (MODE == kStridedRows) {
    q += begin;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int e = j * team + lane;
      f[j] = e < n ? opt_widen<T>(q[e]) : 0.0f;
    }
    return;
  }
  const long long first = (MODE == kWholeRows ? begin : begin & ~7ll) + lane * 8, end = begin + n;
  if (MODE == kWholeRows ? lane * 8 < n : first >= begin && first + 8 <= end) {
    Raw8<T> r;
    r.load(q + first);
    r.pairs(out);
  } else if (MODE == kGroupedRows && first < end && first + 8 > begin) {
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = first + j >= begin && first + j < end ? opt_widen<T>(q[first + j]) : 0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = 0.0f;
  }
}

template <RowMode MODE, typename T>
__device__ __forceinline__ void row_store(void* base, long long begin, int n, int lane, int team, const float2* in) {
  T* q = reinterpret_cast<T*>(base);
  const float* f = reinterpret_cast<const float*>(in);
  if (MODE == kStridedRows) {
    q += begin;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int e = j * team + lane;
      if (e < n) q[e] = opt_narrow<T>(f[j]);
    }
    return;
  }
  const long long first = (MODE == kWholeRows ? begin : begin & ~7ll) + lane * 8, end = begin + n;
  if (MODE == kWholeRows ? lane * 8 < n : first >= begin && first + 8 <= end) {
    opt_store8<T>(q + first, in);
  } else if (MODE == kGroupedRows && first < end && first + 8 > begin) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (first + j >= begin && first + j < end) q[first + j] = opt_narrow<T>(f[j]);
  }
}

// Sums of two values over a team.  `part` is not written again before every thread has passed another barrier.
__device__ __forceinline__ float2 team_sum2(float a, float b, float2* part, int team) {
  for (int m = min(team, 32) >> 1; m > 0; m >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, m);
    b += __shfl_xor_sync(0xffffffffu, b, m);
  }
  if (team <= 32) return make_float2(a, b);
  const int lane = threadIdx.x & 31;
  if (lane == 0) part[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  const float2 q = lane < team >> 5 ? part[lane] : make_float2(0.0f, 0.0f);
  a = q.x, b = q.y;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, m);
    b += __shfl_xor_sync(0xffffffffu, b, m);
  }
  return make_float2(a, b);
}

// What a thread of whole rows reads, as it lies in memory.
template <typename W, typename G>
struct RowRaw {
  Raw8<W> p;
  Raw8<G> g;
  Raw8<float> m, v;

  __device__ __forceinline__ void load(const OptTensor& t, bool master, long long first) {
    p.load(reinterpret_cast<const W*>(master ? t.master : t.param) + first);
    g.load(reinterpret_cast<const G*>(t.grad) + first);
    m.load(reinterpret_cast<const float*>(t.exp_avg) + first);
    v.load(reinterpret_cast<const float*>(t.exp_avg_sq) + first);
  }
};

// Sums are held in 32 bits.  A sum of squares below this has lost more than 2^-27 of itself to terms that vanished: the row, shorter
// than 2^-55, counts as a row of zeros, which has no direction to project on and no length to divide by.  A row whose
// squares overflow, longer than 2^64, is left as it was, with its moments: divided by an infinite length it would
// become zeros.  (An infinity in the row or its gradient makes their product infinite or NaN, and then the row; so does a
// finite gradient whose product with the row passes 2^128.)  Taking such rows again, scaled, is a branch in the
// loop: 131072 rows of 777 bf16 605 instead of 484 us, 29296 of 4096 475 instead of 406.
constexpr float kLeastSquare = 0x1p-110f;

// MOST: threads of a CTA at most.  The registers of a thread (56) are set so that an SM holds two CTAs of up to 576 threads, four
// of up to 288 or nine of 128: 65536 rows of 2304 bf16 (288 threads) take 522 us with room for four or three, 559 with room for
// five, which spills; 77319 of 776 (128 threads) 209, 225 with the registers of three.
// Where an SM holds one CTA, nothing covers its waits, so whole rows of up to 704 threads (80 registers), with 16-bit
// parameters and gradients up to 896 (72), have the next row's loads under way: 60 M bf16 in rows of 5120 / 7168 take 215 /
// 206 us with them and 292 / 260 without; fp32 in rows of 7168 would spill much (356 and 296).  Kernels that spill as they
// are: 4 to 20 bytes in the 704 class with fp32 parameters or with fp32 gradients and masters, in the 896 class and in grouped
// fp32 rows of up to 576 threads; 12 to 48 bytes in all kernels of strided rows.
template <RowMode MODE, typename P, typename G, bool MASTER, int MOST>
__global__ void __launch_bounds__(MOST, MOST <= 576 ? 2 : 1) adamw_unit_rows_kernel(const __grid_constant__ RowArgs a) {
  using W = typename std::conditional<MASTER, float, P>::type;      // type that holds the parameter's value
  __shared__ float2 part[2][32];
  const OptTensor& t = a.t;
  const int team = a.team, teams = blockDim.x / team, slot = threadIdx.x / team, lane = threadIdx.x % team;
  opt_wait();
  OptCoefs co;
  if (!opt_coefs(a.s, co)) return;
  OptCoefs unclipped = co;                            // the gradient is clipped before the projection
  unclipped.clip = 1.0f;
  constexpr bool kAhead = MOST == 704 || MOST == 896;
  RowRaw<W, G> next = {};
  if (kAhead && lane * 8 < a.cols && blockIdx.x < a.rows) next.load(t, MASTER, (long long)blockIdx.x * a.cols + lane * 8);
  for (long long r0 = (long long)blockIdx.x * teams; r0 < a.rows; r0 += (long long)gridDim.x * teams) {
    const long long r = r0 + slot, begin = r * a.cols;
    const int n = r < a.rows ? a.cols : 0;            // past the last row a team only keeps its warp company
    float2 p2[4], g2[4], m2[4], v2[4];
    float *p = reinterpret_cast<float*>(p2), *g = reinterpret_cast<float*>(g2);
    if (kAhead) {
      next.p.pairs(p2), next.g.pairs(g2), next.m.pairs(m2), next.v.pairs(v2);
      if (lane * 8 < a.cols && r0 + gridDim.x < a.rows) next.load(t, MASTER, begin + (long long)gridDim.x * a.cols + lane * 8);
    } else {
      row_load<MODE, W>(MASTER ? t.master : t.param, begin, n, lane, team, p2);
      row_load<MODE, G>(t.grad, begin, n, lane, team, g2);
      row_load<MODE, float>(t.exp_avg, begin, n, lane, team, m2);
      row_load<MODE, float>(t.exp_avg_sq, begin, n, lane, team, v2);
    }
    float gp = 0.0f, pp = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      g[j] *= co.clip;
      gp = fmaf(g[j], p[j], gp);
      pp = fmaf(p[j], p[j], pp);
    }
    const float2 dots = team_sum2(gp, pp, part[0], team);
    const bool wide = dots.y > FLT_MAX && fabsf(dots.x) <= FLT_MAX;
    const float along = dots.y < kLeastSquare ? 0.0f : dots.x / dots.y;      // a NaN passes, here and below
    float len = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) g[j] -= along * p[j];
    adamw_eight(a.s, unclipped, p2, g2, m2, v2);
#pragma unroll
    for (int j = 0; j < 8; j++) len = fmaf(p[j], p[j], len);
    len = team_sum2(len, 0.0f, part[1], team).x;
    const float scale = len < kLeastSquare ? 1.0f : 1.0f / sqrtf(len);      // one division instead of eight: half an ulp more
    const int put = wide || len > FLT_MAX ? 0 : n;
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] *= scale;
    row_store<MODE, P>(t.param, begin, put, lane, team, p2);
    if (MASTER) row_store<MODE, float>(t.master, begin, put, lane, team, p2);
    row_store<MODE, float>(t.exp_avg, begin, put, lane, team, m2);
    row_store<MODE, float>(t.exp_avg_sq, begin, put, lane, team, v2);
  }
  opt_advance(a.s, co.t);
}

constexpr int kRowThreads = 128;      // of a CTA whose rows have a warp or less each
// Rows that do not begin at a group of eight are read in groups from here on (their ends are accesses of
// single elements; bf16: 77220 rows of 777 take 293 us in groups and 330 strided, 131072 of 257 319 and 274).
constexpr int kGroupedFrom = 640;

template <RowMode MODE, typename P, typename G, bool M>
static cudaError_t launch_mode(const RowArgs& a, int threads, cudaStream_t st) {
  auto kernel = threads <= 576 ? adamw_unit_rows_kernel<MODE, P, G, M, 576> : adamw_unit_rows_kernel<MODE, P, G, M, 1024>;
  if constexpr (MODE == kWholeRows) {
    if (threads > 576 && threads <= 704) kernel = adamw_unit_rows_kernel<MODE, P, G, M, 704>;
    if constexpr (sizeof(P) == 2 && sizeof(G) == 2 && !M)
      if (threads > 704 && threads <= 896) kernel = adamw_unit_rows_kernel<MODE, P, G, M, 896>;
  }
  static std::atomic<unsigned> known[33];
  unsigned most = 0;
  if (cudaError_t e = resident_ctas(known[threads / 32], kernel, threads, 32, &most)) return e;
  const long long teams = threads / a.team, ctas = (a.rows + teams - 1) / teams;
  return launch_early(kernel, (unsigned)std::min<long long>(ctas, most), threads, a, st);
}

cudaError_t launch_rows(RowArgs a, int kind, cudaStream_t st) {
  int groups = (a.cols + 7) / 8;      // of eight elements
  RowMode mode = kStridedRows;
  if (a.t.vec && a.cols % 8 == 0) {
    mode = kWholeRows;
  } else if (a.t.vec && a.cols >= kGroupedFrom && (a.cols + 14) / 8 <= 1024) {
    mode = kGroupedRows;
    groups = (a.cols + 14) / 8;       // one more, since a row may begin inside a group
  }
  a.team = 1;
  while (a.team < groups && a.team < 32) a.team *= 2;
  if (groups > 32) a.team = (groups + 31) / 32 * 32;
  const int threads = a.team > 32 ? a.team : kRowThreads;
  cudaError_t e = cudaSuccess;
#define CALL_ROWS(P, G, M)                                                        \
  e = mode == kWholeRows     ? launch_mode<kWholeRows, P, G, M>(a, threads, st)   \
      : mode == kGroupedRows ? launch_mode<kGroupedRows, P, G, M>(a, threads, st) \
                             : launch_mode<kStridedRows, P, G, M>(a, threads, st)
  FLEXSAE_OPT_KINDS(kind, CALL_ROWS)
#undef CALL_ROWS
  t_launches++;
  return e;
}

}  // namespace flexsae
