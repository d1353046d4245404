// The optimizer step behind the decoder losses: norm of all gradients, AdamW with 32-bit or 8-bit
// states over a list of tensors, AdamW on a decoder whose rows are kept at unit length.  The
// reference stops at the gradients (torch-ext/flex_sae/hierarchical_kernels.py:288-299).
//
// Every operator is one pass over its data, bound by HBM: per parameter the step reads the parameter,
// its gradient and two states and writes three of them back (22 bytes with 16-bit weights and 32-bit
// states, 10 bytes with 8-bit states).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <math.h>
#include <new>
#include <type_traits>

#include "flexsae_optim.cuh"

namespace flexsae {

// ---- gradient norm --------------------------------------------------------------------------------------
constexpr int kNormUnits = 4;                               // units of 256 elements a warp takes at a time
constexpr int kNormGrid = 148 * 8;
constexpr int kNormCluster = 8, kNormClusterThreads = 512;
// Elements of a list for which one cluster is enough.  With 2^17 / 2^18 / 2^19 it takes 2.7 / 3.3 / 4.6 us and two launches 3.0 on
// the GPU, but 4.7 and 7.8 us where the host has to keep up.
constexpr int64_t kNormSmall = 1 << 18;
// Tensors of one launch.  What a launch's arguments hold is paid for on the host: a step over 20 tensors takes the
// caller 14 us with room for 32 of them and 23 us with room for 256; the GPU does not notice (3.2 us either way).
constexpr int kSmallBatch = 32, kLargeBatch = 256;

template <int N>
struct NormBatch {
  double* partial;            // one sum per CTA
  float* out;                 // the norm, where one launch is all
  unsigned chunks;
  int count;
  unsigned first[N + 1];
  const void* grad[N];
  long long numel[N];
  unsigned char dtype[N], vec[N];
};

// Sum of eight squares.  The plain 32-bit sum is used where it neither overflowed nor lost terms to
// underflow; otherwise the squares are formed in 64 bits, so that a norm is finite whenever the
// result fits the output.
__device__ __forceinline__ double sum_squares(const float2* pairs) {
  const float* x = reinterpret_cast<const float*>(pairs);
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; j++) s = fmaf(x[j], x[j], s);
  if (s >= 0x1p-90f && s <= FLT_MAX) return (double)s;
  unsigned any = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) any |= __float_as_uint(x[j]) << 1;
  if (!any) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < 8; j++) d = fma((double)x[j], (double)x[j], d);
  return d;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[THREADS / 32];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < THREADS / 32; i++) v += part[i];
  return v;
}

template <typename T>
__device__ __forceinline__ double norm_chunk(const void* grad, long long e0, long long numel, bool aligned, int lane) {
  double acc = 0.0;
  if (aligned && e0 + kNormUnits * kOptBlock <= numel) {
    float2 x[kNormUnits][4];
#pragma unroll
    for (int u = 0; u < kNormUnits; u++) opt_load<T>(grad, e0 + u * kOptBlock, numel, true, lane, 32, x[u]);
#pragma unroll
    for (int u = 0; u < kNormUnits; u++) acc += sum_squares(x[u]);
  } else {
    for (int u = 0; u < kNormUnits; u++) {
      float2 x[4];
      opt_load<T>(grad, e0 + u * kOptBlock, numel, false, lane, 32, x);
      acc += sum_squares(x);
    }
  }
  return acc;
}

// Sum of this thread's share; a CTA takes every gridDim-th chunk of THREADS / 32 warps.
template <int N, int THREADS>
__device__ __forceinline__ double norm_share(const NormBatch<N>& b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double acc = 0.0;
  int i = 0;
  for (unsigned c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    while (c >= b.first[i + 1]) i++;
    const long long e0 = ((long long)(c - b.first[i]) * (THREADS / 32) + warp) * (kNormUnits * kOptBlock);
    if (e0 >= b.numel[i]) continue;
    if (b.dtype[i] == FLEXSAE_F32)
      acc += norm_chunk<float>(b.grad[i], e0, b.numel[i], b.vec[i], lane);
    else if (b.dtype[i] == FLEXSAE_BF16)
      acc += norm_chunk<__nv_bfloat16>(b.grad[i], e0, b.numel[i], b.vec[i], lane);
    else
      acc += norm_chunk<__half>(b.grad[i], e0, b.numel[i], b.vec[i], lane);
  }
  return acc;
}

template <int N>
__global__ void __launch_bounds__(kOptThreads) grad_norm_kernel(const __grid_constant__ NormBatch<N> b) {
  opt_wait();
  const double sum = block_sum<kOptThreads>(norm_share<N, kOptThreads>(b));
  if (threadIdx.x == 0) b.partial[blockIdx.x] = sum;
}

struct NormFinish {
  const double* partial;
  int n;
  float* out;
};

__global__ void __launch_bounds__(kOptThreads) grad_norm_finish_kernel(const NormFinish f) {
  opt_wait();
  double acc = 0.0;
  for (int i = threadIdx.x; i < f.n; i += kOptThreads) acc += f.partial[i];
  acc = block_sum<kOptThreads>(acc);
  if (threadIdx.x == 0) *f.out = (float)sqrt(acc);
}

// Small lists in one launch without a workspace: the CTAs of one cluster leave their sums in the shared memory
// of its first one.  A toy model of 66 k gradients, whose norm is all latency, takes 4.5 us; with two launches it took 8.6.
__global__ void __cluster_dims__(kNormCluster, 1, 1) __launch_bounds__(kNormClusterThreads)
    grad_norm_small_kernel(const __grid_constant__ NormBatch<kSmallBatch> b) {
  namespace cg = cooperative_groups;
  __shared__ double sums[kNormCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                                 // a CTA's shared memory may be written once it runs
  opt_wait();
  const double sum = block_sum<kNormClusterThreads>(norm_share<kSmallBatch, kNormClusterThreads>(b));
  cluster.barrier_wait();
  if (threadIdx.x == 0) cluster.map_shared_rank(sums, 0)[cluster.block_rank()] = sum;
  cluster.sync();
  if (cluster.block_rank() == 0 && threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kNormCluster; i++) total += sums[i];
    *b.out = (float)sqrt(total);
  }
}

// ---- AdamW, 32-bit states -----------------------------------------------------------------------------
// Bound by HBM: 302 M bf16 parameters in 1.03 ms (99 % of the measured copy rate), 268 M fp32 in 1.13 ms (102 %); not
// aligned to eight elements, where single elements are moved, 100 M bf16 take 446 instead of 340 us and fp32 448 instead of 421.
constexpr int kAdamwThreads = 128, kAdamw8Threads = 256;

// The chunks of all tensors (a unit for every one of a CTA's warps) are dealt out to the CTAs in turn.  Step is told about
//   full(first, end, stride)  its complete, aligned chunks of a tensor, which lie in one span of 2^31 elements;
//                             answers the first one that it has not done (for this warp), from which on units go to
//   part(unit)                which does any unit, for the whole warp.
template <int N, typename Step>
__device__ __forceinline__ void opt_walk(const OptBatch<N>& b, Step& step) {
  constexpr int kChunk = Step::kThreads * 8;
  constexpr unsigned kSpan = (1u << 31) / kChunk;
  int i = 0;
  for (unsigned c = blockIdx.x; c < b.chunks;) {
    i = opt_find<N>(b, c, i);
    const OptTensor& t = b.t[i];
    const unsigned first = b.first[i], last = b.first[i + 1];
    step.tensor(t);
    const unsigned whole = t.vec ? (unsigned)(t.numel / kChunk) : 0u;
    unsigned rest = c - first;
    while (rest < whole) {
      const unsigned end = min(whole, (rest / kSpan + 1) * kSpan);
      rest = step.full(rest, end, gridDim.x);
      if (rest < end) break;
    }
    for (; rest < last - first; rest += gridDim.x) {
      const unsigned u = rest * (Step::kThreads / 32) + (threadIdx.x >> 5);
      if ((long long)u * kOptBlock < t.numel) step.part(u);
    }
    c += ((last - 1 - c) / gridDim.x + 1) * gridDim.x;
  }
}

template <typename P, typename G, bool MASTER>
struct AdamwStep {
  static constexpr int kThreads = kAdamwThreads;
  using W = typename std::conditional<MASTER, float, P>::type;      // type that holds the parameter's value
  const OptScalars& s;
  const OptCoefs& co;
  const OptTensor* t;

  __device__ __forceinline__ void tensor(const OptTensor& x) { t = &x; }

  // Elements e0 + lane * 8 ... of a team of `lanes` threads, or every lanes-th of them.
  __device__ __forceinline__ void unit(long long e0, bool vec, int lane, int lanes) const {
    float2 p[4], g[4], m[4], v[4];
    opt_load<W>(MASTER ? t->master : t->param, e0, t->numel, vec, lane, lanes, p);
    opt_load<G>(t->grad, e0, t->numel, vec, lane, lanes, g);
    opt_load<float>(t->exp_avg, e0, t->numel, vec, lane, lanes, m);
    opt_load<float>(t->exp_avg_sq, e0, t->numel, vec, lane, lanes, v);
    adamw_eight(s, co, p, g, m, v);
    opt_store<P>(t->param, e0, t->numel, vec, lane, lanes, p);
    if (MASTER) opt_store<float>(t->master, e0, t->numel, vec, lane, lanes, p);
    opt_store<float>(t->exp_avg, e0, t->numel, vec, lane, lanes, m);
    opt_store<float>(t->exp_avg_sq, e0, t->numel, vec, lane, lanes, v);
  }

  __device__ __forceinline__ unsigned full(unsigned c, unsigned end, unsigned stride) const {
    for (; c < end; c += stride) unit((long long)c * (kThreads * 8), true, threadIdx.x, kThreads);
    return c;
  }
  __device__ __forceinline__ void part(unsigned u) const { unit((long long)u * kOptBlock, false, threadIdx.x & 31, 32); }
};

template <typename P, typename G, bool MASTER, int N>
__global__ void __launch_bounds__(kAdamwThreads, 4) adamw_kernel(const __grid_constant__ OptBatch<N> b) {
  opt_wait();
  OptCoefs co;
  if (!opt_coefs(b.s, co)) return;
  AdamwStep<P, G, MASTER> step{b.s, co, nullptr};
  opt_walk<N>(b, step);
  opt_advance(b.s, co.t);
}

// ---- AdamW, 8-bit states --------------------------------------------------------------------------------
// m is held as e4m3 and v as e5m2, each times one 32-bit scale per 256 elements.  Both are rounded at
// random between their two neighbours: with b2 = 0.999 a step changes v by about 0.1 %, far less than
// half the spacing of an 8-bit float, so that rounding to nearest would never move it; rounding upwards
// with the probability (v - lower) / (upper - lower) keeps the average right.  Adding random bits
// below the last kept one and cutting off does exactly that on the bit pattern of a 32-bit float whose
// exponent has been moved to the small format's, subnormals included (they become 32-bit subnormals).
constexpr float kScaleM = (float)((1.0 / 448.0) * (1.0 + 0x1p-20));     // the largest value stays below the format's last
constexpr float kScaleV = (float)((1.0 / 57344.0) * (1.0 + 0x1p-20));

__device__ __forceinline__ unsigned code_e4m3(float x, float inverse, unsigned random20) {
  const unsigned b = __float_as_uint(__fmul_rn(__fmul_rn(x, inverse), 0x1p-120f));
  return (((b & 0x7fffffffu) + random20) >> 20) | ((b >> 24) & 0x80u);
}

constexpr unsigned kLeastV = 1u << 21;     // the code 1

// v never becomes zero beside larger values: it is at least the format's smallest number (2^-32 of the
// block's largest value), so an element is not divided by its eps alone because its neighbours are large.
__device__ __forceinline__ unsigned code_e5m2(float x, float inverse, unsigned random21) {
  const float y = fmaxf(__fmul_rn(__fmul_rn(x, inverse), 0x1p-112f), __uint_as_float(kLeastV));
  return (__float_as_uint(y) + random21) >> 21;
}

__device__ __forceinline__ float scale_of(unsigned largest, float factor) {
  const float s = __fmul_rn(__uint_as_float(largest), factor);
  return s >= FLT_MIN ? s : 0.0f;
}
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.0f ? __frcp_rn(scale) : 0.0f; }

// Two e4m3 / e5m2 codes, widened.  An e5m2 code is the upper half of a 16-bit float.
__device__ __forceinline__ float2 widen_e4m3x2(unsigned two) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
}
__device__ __forceinline__ float2 widen_e5m2x2(unsigned halves) { return __half22float2(*reinterpret_cast<const __half2*>(&halves)); }

// max(|a|, |b|, |c|), NaN if one of them is
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }

// (x << SHIFT) + y.  Written as instructions: with both summands shifted in C++, the compiler (12.9) dropped the shift in
// one arrangement of the code that follows.
template <int SHIFT>
__device__ __forceinline__ unsigned shift_add(unsigned x, unsigned y) {
  unsigned d;
  asm("{.reg .b32 t; shl.b32 t, %1, %2; add.u32 %0, t, %3;}" : "=r"(d) : "r"(x), "n"(SHIFT), "r"(y));
  return d;
}

// Top bytes of four words, lowest first.
__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// The step, to the same bits as Adamw8Step, for a unit that is cut off, not aligned (all of a tensor's units, if one of its
// pointers is not: 100 M bf16 parameters 516 instead of 180 us, since every access moves one element, every element has a hash
// of its own and no unit is on its way while another is worked on), or holds an infinity or NaN, which
// keep to their own elements: the scale is that of the others (e4m3 has no infinity: a NaN stands for it).  With an eps below kLeastEps, for which the
// approximate root is not good enough, all units come here.
template <typename P, typename G, bool MASTER>
__device__ __forceinline__ void adamw8_part(const OptScalars& s, const OptCoefs& co, const OptTensor* t, unsigned key, unsigned u) {
  using W = typename std::conditional<MASTER, float, P>::type;
  const int lane = threadIdx.x & 31;
  const long long e0 = (long long)u * kOptBlock;
  const int n = (int)min((long long)kOptBlock, t->numel - e0);
  unsigned char* m8 = reinterpret_cast<unsigned char*>(t->exp_avg) + e0;
  unsigned char* v8 = reinterpret_cast<unsigned char*>(t->exp_avg_sq) + e0;
  const float sm = t->exp_avg_scale[u], sv = t->exp_avg_sq_scale[u];
  float2 p[4], g[4], m[4], v[4];
  opt_load<W>(MASTER ? t->master : t->param, e0, t->numel, false, lane, 32, p);
  opt_load<G>(t->grad, e0, t->numel, false, lane, 32, g);
  float* ms = reinterpret_cast<float*>(m);
  float* vs = reinterpret_cast<float*>(v);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int e = j * 32 + lane;
    ms[j] = __fmul_rn(widen_e4m3x2(e < n ? m8[e] : 0u).x, sm);
    vs[j] = __fmul_rn(widen_e5m2x2(e < n ? v8[e] << 8 : 0u).x, sv);
  }
  adamw_eight(s, co, p, g, m, v);
  float top_m = 0.0f, top_v = 0.0f;
  bool overflow = false;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    if (finite(ms[j])) top_m = fmaxf(top_m, fabsf(ms[j]));
    if (finite(vs[j])) top_v = fmaxf(top_v, vs[j]);
    overflow |= vs[j] > FLT_MAX;
  }
  opt_store<P>(t->param, e0, t->numel, false, lane, 32, p);
  if (MASTER) opt_store<float>(t->master, e0, t->numel, false, lane, 32, p);
  const float new_sm = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m)), kScaleM);
  float new_sv = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)), kScaleV);
  if (__any_sync(0xffffffffu, overflow) && new_sv == 0.0f) new_sv = FLT_MIN;      // an infinity times it is one again
  const float im = inverse_of(new_sm), iv = inverse_of(new_sv);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int e = j * 32 + lane;
    if (e >= n) continue;
    const unsigned h = opt_mix((u * (kOptBlock / 2) + (e >> 1)) ^ (key + (u >> 25)));
    m8[e] = (unsigned char)(finite(ms[j]) ? code_e4m3(ms[j], im, e & 1 ? h & 0xfffffu : h >> 12) : 0x7fu);
    v8[e] = (unsigned char)(finite(vs[j]) ? code_e5m2(vs[j], iv, e & 1 ? h >> 11 : h & 0x1fffffu) : vs[j] > FLT_MAX ? 0x7cu : 0x7fu);
  }
  if (lane == 0) {
    t->exp_avg_scale[u] = new_sm;
    t->exp_avg_sq_scale[u] = new_sv;
  }
}

// The 32-bit form has 22 bytes of traffic per element to hide its arithmetic behind, this one 10: at HBM
// speed an SM may spend about 49 instructions on an element; the kernel takes 43.5, and 302 M bf16 parameters
// 0.59 ms, 79 % of the HBM rate (0.78 ms and 96 % with fp32 parameters).  So the arithmetic is in packed pairs,
// root and reciprocal are the approximate ones (2 u each; they only reach the parameter), the codes are
// formed in the top byte of a word, where shift and random bits are one addition, one hash serves a
// pair of elements, and a warp's next unit is on its way while it works on one.
template <typename P, typename G, bool MASTER>
struct Adamw8Step {
  static constexpr int kThreads = kAdamw8Threads;
  using W = typename std::conditional<MASTER, float, P>::type;      // type that holds the parameter's value
  struct Raw {
    Raw8<W> p;
    Raw8<G> g;
    Raw8<unsigned char> m, v;
    float sm, sv;
  };
  const OptScalars& s;
  const OptCoefs& co;
  const OptTensor* t;
  unsigned key;

  __device__ __forceinline__ void tensor(const OptTensor& x) {
    t = &x;
    key = opt_key(s.seed, co.t, x.index);
  }

  // Where this thread's eight elements of a chunk begin, and its warp's scales.
  struct Place {
    const W* w;
    P* p;
    const G* g;
    unsigned char *m, *v;
    float *sm, *sv;
    unsigned pair, high;      // half the element's index: low 32 bits, and the key with the high ones
  };

  // `e` elements on from the place: 32 bits are enough, and one instruction makes an address.
  __device__ __forceinline__ static void fetch(const Place& at, unsigned e, Raw& r) {
    r.p.load(at.w + e);
    r.g.load(at.g + e);
    r.m.load(at.m + e);
    r.v.load(at.v + e);
    r.sm = at.sm[e / kOptBlock];
    r.sv = at.sv[e / kOptBlock];
  }

  __device__ __forceinline__ unsigned full(unsigned c, unsigned end, unsigned stride) const {
    const size_t e0 = (size_t)c * (kThreads * 8) + threadIdx.x * 8;
    Place at;
    at.p = reinterpret_cast<P*>(t->param) + e0;
    at.w = MASTER ? reinterpret_cast<const W*>(t->master + e0) : reinterpret_cast<const W*>(at.p);
    at.g = reinterpret_cast<const G*>(t->grad) + e0;
    at.m = reinterpret_cast<unsigned char*>(t->exp_avg) + e0;
    at.v = reinterpret_cast<unsigned char*>(t->exp_avg_sq) + e0;
    at.sm = t->exp_avg_scale + e0 / kOptBlock;
    at.sv = t->exp_avg_sq_scale + e0 / kOptBlock;
    at.pair = (unsigned)(e0 / 2);
    at.high = key + (unsigned)(e0 >> 33);
    Raw next;
    fetch(at, 0, next);
    unsigned e = 0;
    for (; c < end; c += stride, e += stride * (kThreads * 8)) {
      const Raw now = next;
      if (c + stride < end) fetch(at, e + stride * (kThreads * 8), next);
      if (!unit(now, at, e)) break;
    }
    return c;
  }

  // False: the unit holds an infinity or NaN, and nothing was written.
  __device__ __forceinline__ bool unit(const Raw& r, const Place& at, unsigned e) const {
    float2 p[4], g[4], m[4], v[4];
    m[0] = widen_e4m3x2(r.m.w.x & 0xffffu), m[1] = widen_e4m3x2(r.m.w.x >> 16);
    m[2] = widen_e4m3x2(r.m.w.y & 0xffffu), m[3] = widen_e4m3x2(r.m.w.y >> 16);
    v[0] = widen_e5m2x2(__byte_perm(r.v.w.x, 0, 0x1404)), v[1] = widen_e5m2x2(__byte_perm(r.v.w.x, 0, 0x3424));
    v[2] = widen_e5m2x2(__byte_perm(r.v.w.y, 0, 0x1404)), v[3] = widen_e5m2x2(__byte_perm(r.v.w.y, 0, 0x3424));
    r.g.pairs(g);
    float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      m[j] = mul2(m[j], both(r.sm));
      v[j] = mul2(v[j], both(r.sv));
      moments_pair(s, co.clip, g[j], m[j], v[j]);
      top_m = max_abs3(top_m, m[j].x, m[j].y);
      top_v = max_abs3(top_v, v[j].x, v[j].y);
    }
    const unsigned largest_m = __reduce_max_sync(0xffffffffu, __float_as_uint(top_m));
    const unsigned largest_v = __reduce_max_sync(0xffffffffu, __float_as_uint(top_v));
    if (max(largest_m, largest_v) >= 0x7f800000u) return false;
    r.p.pairs(p);
#pragma unroll
    for (int j = 0; j < 4; j++) p[j] = param_pair(s, co, p[j], m[j], v[j]);
    opt_store8<P>(at.p + e, p);
    if (MASTER) opt_store8<float>(reinterpret_cast<float*>(const_cast<W*>(at.w)) + e, p);
    const float new_sm = scale_of(largest_m, kScaleM), new_sv = scale_of(largest_v, kScaleV);
    const float2 im = both(inverse_of(new_sm)), iv = both(inverse_of(new_sv));
    // element 2 j takes bits 12..31 of the pair's hash for m and 0..20 for v, element 2 j + 1 bits 0..19 and
    // 11..31: as 24 bits under the top byte that is h >> 8 for two of them.  The first step of the hash is
    // the same for the four pairs of a lane but for their last two bits.
    const unsigned x = (at.pair + e / 2) ^ at.high;
    unsigned qm[8], qv[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const unsigned h = opt_mix_rest((x ^ x >> 16) ^ j);
      const float2 ym = mul2(mul2(m[j], im), both(0x1p-120f));
      const float2 yv = mul2(mul2(v[j], iv), both(0x1p-112f));
      const unsigned m0 = __float_as_uint(ym.x), m1 = __float_as_uint(ym.y);
      const unsigned v0 = __float_as_uint(fmaxf(yv.x, __uint_as_float(kLeastV))), v1 = __float_as_uint(fmaxf(yv.y, __uint_as_float(kLeastV)));
      qm[2 * j] = shift_add<4>(m0, h >> 8) | (m0 & 0x80000000u);
      qm[2 * j + 1] = shift_add<4>(m1, h << 4 & 0xffffffu) | (m1 & 0x80000000u);
      qv[2 * j] = shift_add<3>(v0, h << 3 & 0xffffffu);
      qv[2 * j + 1] = shift_add<3>(v1, h >> 8);
    }
    Raw8<unsigned char> cm, cv;
    cm.w = make_uint2(top_bytes(qm[0], qm[1], qm[2], qm[3]), top_bytes(qm[4], qm[5], qm[6], qm[7]));
    cv.w = make_uint2(top_bytes(qv[0], qv[1], qv[2], qv[3]), top_bytes(qv[4], qv[5], qv[6], qv[7]));
    cm.store(at.m + e);
    cv.store(at.v + e);
    if (threadIdx.x % 32 == 0) {
      at.sm[e / kOptBlock] = new_sm;
      at.sv[e / kOptBlock] = new_sv;
    }
    return true;
  }

  __device__ __forceinline__ void part(unsigned u) const { adamw8_part<P, G, MASTER>(s, co, t, key, u); }
};

template <typename P, typename G, bool MASTER, int N>
__global__ void __launch_bounds__(kAdamw8Threads, sizeof(P) == 4 || sizeof(G) == 4 || MASTER ? 2 : 3) adamw8_kernel(const __grid_constant__ OptBatch<N> b) {
  opt_wait();
  OptCoefs co;
  if (!opt_coefs(b.s, co)) return;
  Adamw8Step<P, G, MASTER> step{b.s, co, nullptr, 0};
  opt_walk<N>(b, step);
  opt_advance(b.s, co.t);
}

// ---- host side ---------------------------------------------------------------------------------------------
constexpr int64_t kOptMaxTensors = 1 << 16;
constexpr int64_t kOptMaxNumel = 1ll << 38;
constexpr unsigned long long kOptMaxChunks = 1ull << 30;
// Elements of a list in all (a tensor may be in it many times): fewer than 2^30 chunks, so a launch takes as many tensors as it
// has room for, which the workspace counts on.
constexpr int64_t kNormMaxElements = 1ll << 42;
// A stretch of memory that a step reads or writes.
struct Stretch {
  uintptr_t begin, end;
  bool written;
};

static int check_scalars(const int64_t* step, double lr, double beta1, double beta2, double eps, double weight_decay,
                         const float* norm, double max_norm) {
  if (!step) return fail(FLEXSAE_EINVAL, "null pointer argument: step");
  if (!aligned(step, 8)) return fail(FLEXSAE_EINVAL, "step must be 8-byte aligned");
  if (!(lr >= 0.0 && lr <= FLT_MAX)) return fail(FLEXSAE_EINVAL, "lr = %g is not a finite number >= 0", lr);
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return fail(FLEXSAE_EINVAL, "betas %g, %g outside [0, 1)", beta1, beta2);
  if (!(eps >= FLT_MIN && eps <= FLT_MAX)) return fail(FLEXSAE_EINVAL, "eps = %g must be a normal 32-bit number > 0", eps);
  if (!(weight_decay >= 0.0 && weight_decay <= FLT_MAX)) return fail(FLEXSAE_EINVAL, "weight_decay = %g is not a finite number >= 0", weight_decay);
  if (norm && !(max_norm > 0.0)) return fail(FLEXSAE_EINVAL, "max_norm = %g must be positive", max_norm);
  return 0;
}

static OptScalars make_scalars(int64_t* step, double lr, const float* lr_device, double beta1, double beta2, double eps,
                               double weight_decay, const float* norm, double max_norm, uint32_t seed) {
  OptScalars s;
  s.step = reinterpret_cast<unsigned long long*>(step);
  s.norm = norm;
  s.lr_device = lr_device;
  s.lr = lr;
  s.weight_decay = weight_decay;
  s.log_beta1 = log(beta1);
  s.log_beta2 = log(beta2);
  s.beta1 = (float)beta1;
  s.one_minus_beta1 = (float)(1.0 - beta1);
  s.beta2 = (float)beta2;
  s.one_minus_beta2 = (float)(1.0 - beta2);
  s.eps = (float)eps;
  s.max_norm = (float)max_norm;
  s.minus_zero = -0.0f;
  s.seed = seed;
  s.advance = 0;
  return s;
}

// Checks one tensor's description and notes the memory that it reads and writes.
static int check_tensor(const flexsae_optim_tensor& t, int64_t i, int state_bits, bool rows, Stretch* out, int* used) {
  const long long at = (long long)i;
  if (!opt_dtype(t.param_dtype)) return fail(FLEXSAE_EINVAL, "tensor %lld: unknown dtype code %d", at, t.param_dtype);
  if (t.grad_dtype != t.param_dtype && t.grad_dtype != FLEXSAE_F32)
    return fail(FLEXSAE_EINVAL, "tensor %lld: the gradient's type (code %d) must be the parameter's or fp32", at, t.grad_dtype);
  if (t.master && t.param_dtype == FLEXSAE_F32) return fail(FLEXSAE_EINVAL, "tensor %lld: a master copy goes with 16-bit parameters only", at);
  if (t.numel < 0 || t.numel > kOptMaxNumel) return fail(FLEXSAE_EINVAL, "tensor %lld: numel %lld outside [0, 2^38]", at, (long long)t.numel);
  *used = 0;
  if (t.numel == 0) return 0;
  if (rows) {
    if (t.cols < 1 || t.numel % t.cols) return fail(FLEXSAE_EINVAL, "tensor %lld: %lld elements are not rows of %lld", at, (long long)t.numel, (long long)t.cols);
    if (t.cols > kOptMaxRow) return fail(FLEXSAE_EUNSUPPORTED, "tensor %lld: rows of %lld elements, at most %d are supported", at, (long long)t.cols, kOptMaxRow);
  }
  if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(FLEXSAE_EINVAL, "tensor %lld: null pointer argument", at);
  const size_t n = (size_t)t.numel, ps = opt_size(t.param_dtype), gs = opt_size(t.grad_dtype), ss = state_bits == 8 ? 1 : 4;
  const size_t scales = state_bits == 8 ? (n + kOptBlock - 1) / kOptBlock * 4 : 0;
  if (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return fail(FLEXSAE_EINVAL, "tensor %lld: null pointer argument: scales", at);
  const struct { const void* p; size_t bytes, align; bool written; } use[] = {
      {t.param, n * ps, ps, true}, {t.grad, n * gs, gs, false}, {t.exp_avg, n * ss, ss, true}, {t.exp_avg_sq, n * ss, ss, true},
      {t.master, t.master ? n * 4 : 0, 4, true}, {t.exp_avg_scale, scales, 4, true}, {t.exp_avg_sq_scale, scales, 4, true}};
  for (const auto& u : use) {
    if (!u.bytes) continue;
    if (!aligned(u.p, u.align)) return fail(FLEXSAE_EINVAL, "tensor %lld: a pointer is not aligned to its elements", at);
    const uintptr_t b = reinterpret_cast<uintptr_t>(u.p);
    out[(*used)++] = Stretch{b, b + u.bytes, u.written};
  }
  return 0;
}

// Tensors given twice, states that overlap: two CTAs would write the same memory.
static int check_overlap(Stretch* s, int64_t n) {
  std::sort(s, s + n, [](const Stretch& a, const Stretch& b) { return a.begin < b.begin; });
  uintptr_t end = 0, end_written = 0;
  for (int64_t i = 0; i < n; i++) {
    if (s[i].begin < end_written || (s[i].written && s[i].begin < end))
      return fail(FLEXSAE_EINVAL, "a tensor is given twice, or two of the tensors (or one and the step word, lr or norm) overlap in memory");
    end = std::max(end, s[i].end);
    if (s[i].written) end_written = std::max(end_written, s[i].end);
  }
  return 0;
}

static int check_tensors(const flexsae_optim_tensor* t, int64_t n, int state_bits, bool rows, const int64_t* step, const float* lr_device,
                         const float* norm) {
  if (n < 0 || n > kOptMaxTensors) return fail(FLEXSAE_EINVAL, "%lld tensors, between 0 and %lld are supported", (long long)n, (long long)kOptMaxTensors);
  if (n > 0 && !t) return fail(FLEXSAE_EINVAL, "null pointer argument: tensors");
  Stretch few[7 * kSmallBatch + 3];
  Stretch* all = n <= kSmallBatch ? few : new (std::nothrow) Stretch[7 * n + 3];
  if (!all) return fail(FLEXSAE_EINVAL, "out of host memory");
  int64_t used = 0;
  const struct { const void* p; size_t bytes; bool written; } words[] = {{step, 8, true}, {lr_device, 4, false}, {norm, 4, false}};
  for (const auto& w : words) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(w.p);
    if (w.p) all[used++] = Stretch{b, b + w.bytes, w.written};
  }
  int rc = 0;
  for (int64_t i = 0; i < n && rc == 0; i++) {
    int k = 0;
    rc = check_tensor(t[i], i, state_bits, rows, all + used, &k);
    used += k;
  }
  if (rc == 0) rc = check_overlap(all, used);
  if (all != few) delete[] all;
  return rc;
}

// What the loads of one SM have under way at most in the 32-bit step, which sets how many CTAs it is given.
// More costs HBM throughput: 302 M bf16 parameters take 1.10 / 1.03 / 1.08 ms with 3 / 4 / 5 CTAs of 12 KB
// each, 268 M fp32 parameters 1.25 / 1.12 / 1.18 ms with 2 / 3 / 4 of 16 KB.
constexpr int kBytesInFlight = 48 * 1024;

template <int N>
static cudaError_t launch_adamw(const OptBatch<N>& b, int kind, int state_bits, cudaStream_t st) {
  const unsigned ctas = std::max(1u, b.chunks);
  cudaError_t e = cudaSuccess;
  unsigned most = 0;
#define CALL_ADAMW(P, G, M)                                                                                  \
  {                                                                                                          \
    static std::atomic<unsigned> known[2];                                                                   \
    if (state_bits == 8) {                                                                                   \
      const auto kernel = adamw8_kernel<P, G, M, N>;                                                         \
      e = resident_ctas(known[1], kernel, kAdamw8Threads, 32, &most);                                        \
      if (e == cudaSuccess) e = launch_early(kernel, std::min(ctas, most), kAdamw8Threads, b, st);           \
    } else {                                                                                                 \
      constexpr int bytes = 8 * ((M ? 4 : sizeof(P)) + sizeof(G) + 8);                                       \
      const auto kernel = adamw_kernel<P, G, M, N>;                                                          \
      e = resident_ctas(known[0], kernel, kAdamwThreads, kBytesInFlight / (kAdamwThreads * bytes), &most);   \
      if (e == cudaSuccess) e = launch_early(kernel, std::min(ctas, most), kAdamwThreads, b, st);            \
    }                                                                                                        \
  }
  FLEXSAE_OPT_KINDS(kind, CALL_ADAMW)
#undef CALL_ADAMW
  t_launches++;
  return e;
}

// Launches the tensors ids[0..n) of one kind, at most N at a time.
template <int N>
static cudaError_t run_kind(const flexsae_optim_tensor* t, const int* ids, int n, int kind, int state_bits, const OptScalars& s,
                            bool last_kind, cudaStream_t st) {
  int k = 0;
  do {
    OptBatch<N> b;
    b.s = s;
    b.count = 0;
    unsigned long long chunks = 0;
    b.first[0] = 0;
    while (k < n && b.count < N) {
      OptTensor d = make_tensor(t[ids[k]], ids[k], state_bits);
      if (state_bits == 8 && s.eps < kLeastEps) d.vec = 0;
      const unsigned long long chunk = 8 * (state_bits == 8 ? kAdamw8Threads : kAdamwThreads);
      const unsigned long long c = ((unsigned long long)d.numel + chunk - 1) / chunk;
      if (b.count && chunks + c > kOptMaxChunks) break;
      chunks += c;
      b.t[b.count++] = d;
      b.first[b.count] = (unsigned)chunks;
      k++;
    }
    b.chunks = (unsigned)chunks;
    b.s.advance = last_kind && k == n;
    if (cudaError_t e = launch_adamw<N>(b, kind, state_bits, st)) return e;
  } while (k < n);
  return cudaSuccess;
}

static int adamw_impl(const flexsae_optim_tensor* t, int64_t n, int state_bits, const OptScalars& s, cudaStream_t st) {
  // positions of the non-empty tensors, kind by kind
  int few[kSmallBatch];
  int* ids = n <= kSmallBatch ? few : new (std::nothrow) int[n];
  if (!ids) return fail(FLEXSAE_EINVAL, "out of host memory");
  int begin[kOptKinds + 1], used = 0, last = 0;
  for (int kind = 0; kind < kOptKinds; kind++) {
    begin[kind] = used;
    for (int64_t i = 0; i < n; i++)
      if (t[i].numel > 0 && kind_of(t[i]) == kind) ids[used++] = (int)i;
    if (used > begin[kind]) last = kind;
  }
  begin[kOptKinds] = used;
  cudaError_t e = cudaSuccess;
  for (int kind = 0; kind <= last && e == cudaSuccess; kind++) {
    const int m = begin[kind + 1] - begin[kind];
    if (m == 0 && !(kind == last && used == 0)) continue;      // nothing to update: one launch still counts the step
    e = m <= kSmallBatch ? run_kind<kSmallBatch>(t, ids + begin[kind], m, kind, state_bits, s, kind == last, st)
                         : run_kind<kLargeBatch>(t, ids + begin[kind], m, kind, state_bits, s, kind == last, st);
  }
  if (ids != few) delete[] ids;
  if (e != cudaSuccess) return fail((int)e, "AdamW launch failed: %s", cudaGetErrorString(e));
  return 0;
}

template <int N>
static cudaError_t launch_norm(const NormBatch<N>& b, unsigned grid, cudaStream_t st) {
  t_launches++;
  return launch_early(grad_norm_kernel<N>, grid, kOptThreads, b, st);
}

}  // namespace flexsae

using namespace flexsae;

extern "C" {

int flexsae_grad_norm_workspace_bytes(int64_t n, int64_t elements, size_t* bytes) {
  if (n < 0 || n > kOptMaxTensors) return fail(FLEXSAE_EINVAL, "%lld tensors, between 0 and %lld are supported", (long long)n, (long long)kOptMaxTensors);
  if (elements < 0 || elements > kNormMaxElements || !bytes)
    return fail(FLEXSAE_EINVAL, "%lld elements outside [0, 2^42], or null pointer", (long long)elements);
  *bytes = n <= kSmallBatch && elements <= kNormSmall ? 0 : (size_t)((n + kLargeBatch - 1) / kLargeBatch + 1) * kNormGrid * sizeof(double);
  return 0;
}

int flexsae_grad_norm(const void* const* grads_host, const int64_t* numel_host, const int32_t* dtypes_host, int64_t n,
                      float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
  t_launches = 0;
  if (n < 0 || n > kOptMaxTensors) return fail(FLEXSAE_EINVAL, "%lld tensors, between 0 and %lld are supported", (long long)n, (long long)kOptMaxTensors);
  if (!norm_out || (n > 0 && (!grads_host || !numel_host || !dtypes_host))) return fail(FLEXSAE_EINVAL, "null pointer argument");
  if (!aligned(norm_out, 4)) return fail(FLEXSAE_EINVAL, "norm_out must be 4-byte aligned");
  int64_t elements = 0;
  for (int64_t i = 0; i < n; i++) {
    if (!opt_dtype(dtypes_host[i])) return fail(FLEXSAE_EINVAL, "tensor %lld: unknown dtype code %d", (long long)i, dtypes_host[i]);
    if (numel_host[i] < 0 || numel_host[i] > kOptMaxNumel) return fail(FLEXSAE_EINVAL, "tensor %lld: numel %lld outside [0, 2^38]", (long long)i, (long long)numel_host[i]);
    if (numel_host[i] > 0 && !grads_host[i]) return fail(FLEXSAE_EINVAL, "tensor %lld: null pointer argument", (long long)i);
    if (!aligned(grads_host[i], opt_size(dtypes_host[i]))) return fail(FLEXSAE_EINVAL, "tensor %lld: a pointer is not aligned to its elements", (long long)i);
    elements += numel_host[i];
  }
  size_t need = 0;
  if (int rc = flexsae_grad_norm_workspace_bytes(n, elements, &need)) return rc;
  if (need && (!workspace || !aligned(workspace, 8))) return fail(FLEXSAE_EINVAL, "workspace must be given, 8-byte aligned");
  if (workspace_bytes < need) return fail(FLEXSAE_EWORKSPACE, "gradient norm workspace too small: %zu < %zu bytes", workspace_bytes, need);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t i = 0;
  // The next tensors, as many as fit, in chunks of `chunk` elements.
  const auto gather = [&](auto& b, int most, unsigned long long chunk) {
    unsigned long long chunks = 0;
    b.count = 0;
    b.first[0] = 0;
    for (; i < n && b.count < most; i++) {
      const unsigned long long c = ((unsigned long long)numel_host[i] + chunk - 1) / chunk;
      if (c == 0) continue;
      chunks += c;
      b.grad[b.count] = grads_host[i];
      b.numel[b.count] = numel_host[i];
      b.dtype[b.count] = (unsigned char)dtypes_host[i];
      b.vec[b.count] = aligned(grads_host[i], 8 * opt_size(dtypes_host[i]));
      b.first[++b.count] = (unsigned)chunks;
    }
    b.chunks = (unsigned)chunks;
    b.partial = nullptr;
    b.out = norm_out;
  };
  cudaError_t e = cudaSuccess;
  if (!need) {
    NormBatch<kSmallBatch> b;
    gather(b, kSmallBatch, kNormClusterThreads * 8 * kNormUnits);
    e = launch_early(grad_norm_small_kernel, kNormCluster, kNormClusterThreads, b, st);
    t_launches++;
  } else {
    double* partial = reinterpret_cast<double*>(workspace);
    int parts = 0;
    const auto run = [&](auto& b, int most) {
      gather(b, most, kOptThreads * 8 * kNormUnits);
      if (!b.count) return;
      const unsigned grid = std::min(b.chunks, (unsigned)kNormGrid);
      b.partial = partial + parts;
      e = launch_norm(b, grid, st);
      parts += (int)grid;
    };
    while (i < n && e == cudaSuccess) {
      if (n <= kSmallBatch) {
        NormBatch<kSmallBatch> b;
        run(b, kSmallBatch);
      } else {
        NormBatch<kLargeBatch> b;
        run(b, kLargeBatch);
      }
    }
    if (e == cudaSuccess) {
      e = launch_early(grad_norm_finish_kernel, 1, kOptThreads, NormFinish{partial, parts, norm_out}, st);
      t_launches++;
    }
  }
  if (e != cudaSuccess) return fail((int)e, "gradient norm launch failed: %s", cudaGetErrorString(e));
  return 0;
}

int flexsae_adamw_step(const flexsae_optim_tensor* tensors_host, int64_t n, int state_bits, int64_t* step, double lr,
                       const float* lr_device, double beta1, double beta2, double eps, double weight_decay, const float* norm,
                       double max_norm, uint32_t seed, void* stream) {
  t_launches = 0;
  if (state_bits != 32 && state_bits != 8) return fail(FLEXSAE_EINVAL, "states of %d bits: 32 and 8 are supported", state_bits);
  if (int rc = check_scalars(step, lr, beta1, beta2, eps, weight_decay, norm, max_norm)) return rc;
  if (int rc = check_tensors(tensors_host, n, state_bits, false, step, lr_device, norm)) return rc;
  return adamw_impl(tensors_host, n, state_bits,
                    make_scalars(step, lr, lr_device, beta1, beta2, eps, weight_decay, norm, max_norm, seed),
                    reinterpret_cast<cudaStream_t>(stream));
}

int flexsae_adamw_unit_rows_step(const flexsae_optim_tensor* tensors_host, int64_t n, int64_t* step, double lr,
                                 const float* lr_device, double beta1, double beta2, double eps, double weight_decay,
                                 const float* norm, double max_norm, void* stream) {
  t_launches = 0;
  if (int rc = check_scalars(step, lr, beta1, beta2, eps, weight_decay, norm, max_norm)) return rc;
  if (int rc = check_tensors(tensors_host, n, 32, true, step, lr_device, norm)) return rc;
  const OptScalars s = make_scalars(step, lr, lr_device, beta1, beta2, eps, weight_decay, norm, max_norm, 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t last = -1;
  for (int64_t i = 0; i < n; i++)
    if (tensors_host[i].numel > 0) last = i;
  if (last < 0) return adamw_impl(nullptr, 0, 32, s, st);        // nothing to update: the step still counts
  for (int64_t i = 0; i <= last; i++) {
    const flexsae_optim_tensor& t = tensors_host[i];
    if (t.numel == 0) continue;
    RowArgs a;
    a.s = s;
    a.s.advance = i == last;
    a.t = make_tensor(t, i, 32);
    a.rows = t.numel / t.cols;
    a.cols = (int)t.cols;
    if (cudaError_t e = launch_rows(a, kind_of(t), st)) return fail((int)e, "unit-row AdamW launch failed: %s", cudaGetErrorString(e));
  }
  return 0;
}

}  // extern "C"
