// Argument blocks and device helpers of the optimizer kernels (gradient norm, AdamW steps).
//
// All of them stream their tensors once, so the unit of work is the same everywhere: one warp takes
// 256 consecutive elements, eight per lane.  Lane l holds elements 8 l .. 8 l + 7 where every tensor
// involved is aligned for one access per lane (32 bytes for 32-bit elements, 16 for 16-bit, 8 for
// 8-bit ones) and the 256 elements are all there, and elements l, 32 + l, 64 + l, ... otherwise (the
// lanes of a warp then still touch consecutive memory).
#pragma once

#include <cuda_fp8.h>
#include <float.h>

#include <algorithm>
#include <atomic>

#include "flexsae_common.cuh"
#include "flexsae_host.cuh"

namespace flexsae {

constexpr int kOptThreads = 256;
constexpr int kOptBlock = 256;                              // elements of a warp's unit = elements that share one scale
constexpr int kOptMaxRow = 8192;                            // longest row of the unit-row step

// Tensor lists travel as kernel arguments (up to 32764 bytes), so a call needs no copy to the device
// and a captured graph holds its own list.
struct OptTensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  float* master;
  long long numel;
  int index;     // position in the caller's list (part of the random key)
  int vec;       // every pointer allows eight elements in one access
};

struct OptScalars {
  unsigned long long* step;   // steps taken (low 40 bits) and, while a step runs, finished CTAs (high 24 bits)
  const float* norm;          // gradient norm, or NULL
  const float* lr_device;     // learning rate on the device, or NULL
  double lr, weight_decay, log_beta1, log_beta2;
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, max_norm, minus_zero;
  unsigned seed;
  int advance;                // this launch is the last of its step
};

template <int N>
struct OptBatch {
  OptScalars s;
  unsigned chunks;
  int count;
  unsigned first[N + 1];      // first chunk of each tensor
  OptTensor t[N];
};

struct OptCoefs {
  float clip;     // factor of the gradients
  float decay;    // 1 - lr * weight_decay
  float rate;     // lr / (1 - beta1^t)
  float root;     // 1 / sqrt(1 - beta2^t)
  unsigned long long t;
};

constexpr unsigned long long kStepMask = (1ull << 40) - 1;

// Waits until the kernels before this one in the stream have finished and their results can be seen.
__device__ __forceinline__ void opt_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The numbers that are the same for every element of a step.  False: the gradient norm is not finite
// and the step does not take place.  Every thread works them out, in 32 bits from t log b
// on, which is formed in 64 and rounded (1 - b^t is off by at most the same relative error); then come expm1f and a division, or
// a root and a reciprocal, so that rate and root are within 4 u each.
__device__ __forceinline__ bool opt_coefs(const OptScalars& s, OptCoefs& c) {
  c.clip = 1.0f;
  if (s.norm) {
    const float n = *s.norm;
    if (!(fabsf(n) <= FLT_MAX)) return false;
    c.clip = fminf(__fmul_rn(__frcp_rn(__fadd_rn(n, 1e-6f)), s.max_norm), 1.0f);
  }
  c.t = (*reinterpret_cast<volatile unsigned long long*>(s.step) & kStepMask) + 1;
  const double lr = s.lr_device ? (double)*s.lr_device : s.lr;
  const double t = (double)c.t;
  c.decay = (float)(1.0 - lr * s.weight_decay);
  c.rate = __fdiv_rn((float)lr, -expm1f((float)(t * s.log_beta1)));   // 1 - b^t without cancellation
  c.root = __frcp_rn(__fsqrt_rn(-expm1f((float)(t * s.log_beta2))));
  return true;
}

// Every CTA reads the step count when it starts; the last CTA to finish writes the next one, so no CTA
// can see it and no other launch is needed.
__device__ __forceinline__ void opt_advance(const OptScalars& s, unsigned long long t) {
  if (!s.advance) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned long long before = atomicAdd(s.step, kStepMask + 1);
    if ((before >> 40) == gridDim.x - 1) *reinterpret_cast<volatile unsigned long long*>(s.step) = t;
  }
}

// Tensor that owns chunk c, searched upwards from tensor i.
template <int N>
__device__ __forceinline__ int opt_find(const OptBatch<N>& b, unsigned c, int i) {
  if (c < b.first[i + 1]) return i;
  int lo = i + 1, hi = b.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c < b.first[mid + 1]) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// ---- eight elements of a lane ---------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float opt_widen(T x) { return x; }
template <>
__device__ __forceinline__ float opt_widen<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float opt_widen<__half>(__half x) { return __half2float(x); }
// 16-bit parameters are rounded to nearest, as torch's optimizers do: a change below half their spacing is lost unless a
// master copy holds it.
template <typename T>
__device__ __forceinline__ T opt_narrow(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 opt_narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half opt_narrow<__half>(float x) { return __float2half_rn(x); }

// Eight elements of a lane as they lie in memory, moved in one access.  With 32-bit elements that is 32
// bytes a lane: two 16-byte accesses would each touch every sector of the unit and use half of it.  (With the loads
// under way limited as they are, AdamW in fp32, 268 M parameters, takes 1.13 ms either way.)
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
    asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w) : "l"(p));
  }
  __device__ __forceinline__ void store(T* p) const {
    asm volatile("st.global.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(w[0].x), "r"(w[0].y), "r"(w[0].z), "r"(w[0].w) : "memory");
  }
  __device__ __forceinline__ void pairs(float2* f) const { Pack<T>::unpack_pairs(w[0], f); }
  __device__ __forceinline__ void pack(const float2* f) { w[0] = Pack<T>::pack(reinterpret_cast<const float*>(f)); }
};
template <>
__device__ __forceinline__ void Raw8<float>::load(const float* p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w), "=r"(w[1].x), "=r"(w[1].y), "=r"(w[1].z), "=r"(w[1].w)
               : "l"(p));
}
template <>
__device__ __forceinline__ void Raw8<float>::store(float* p) const {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0].x), "r"(w[0].y), "r"(w[0].z),
               "r"(w[0].w), "r"(w[1].x), "r"(w[1].y), "r"(w[1].z), "r"(w[1].w)
               : "memory");
}
template <>
__device__ __forceinline__ void Raw8<float>::pairs(float2* f) const {
  Pack<float>::unpack_pairs(w[0], f);
  Pack<float>::unpack_pairs(w[1], f + 2);
}
template <>
__device__ __forceinline__ void Raw8<float>::pack(const float2* f) {
  w[0] = Pack<float>::pack(reinterpret_cast<const float*>(f));
  w[1] = Pack<float>::pack(reinterpret_cast<const float*>(f + 2));
}
template <>
struct Raw8<unsigned char> {
  uint2 w;
  __device__ __forceinline__ void load(const unsigned char* p) {
    asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(p));
  }
  __device__ __forceinline__ void store(unsigned char* p) const {
    asm volatile("st.global.v2.b32 [%0], {%1,%2};" ::"l"(p), "r"(w.x), "r"(w.y) : "memory");
  }
};

template <typename T>
__device__ __forceinline__ void opt_store8(T* p, const float2* f) {
  Raw8<T> r;
  r.pack(f);
  r.store(p);
}

// `e0` is the first element of the unit, `lane` / `lanes` this thread's place in the team that shares it.
template <typename T>
__device__ __forceinline__ void opt_load(const void* base, long long e0, long long end, bool vec, int lane, int lanes, float2* out) {
  const T* q = reinterpret_cast<const T*>(base) + e0;
  if (vec) {
    Raw8<T> r;
    r.load(q + lane * 8);
    r.pairs(out);
  } else {
    float* f = reinterpret_cast<float*>(out);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int e = j * lanes + lane;
      f[j] = e < end - e0 ? opt_widen<T>(q[e]) : 0.0f;
    }
  }
}

template <typename T>
__device__ __forceinline__ void opt_store(void* base, long long e0, long long end, bool vec, int lane, int lanes, const float2* in) {
  T* q = reinterpret_cast<T*>(base) + e0;
  if (vec) {
    opt_store8<T>(q + lane * 8, in);
  } else {
    const float* f = reinterpret_cast<const float*>(in);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int e = j * lanes + lane;
      if (e < end - e0) q[e] = opt_narrow<T>(f[j]);
    }
  }
}

// The two running averages.  Multiplications and additions are rounded one by one (no fused
// multiply-add), so that the states -- and with them the 8-bit codes -- are the same bits wherever the
// formula is written out in 32-bit arithmetic.
__device__ __forceinline__ void opt_moments(const OptScalars& s, float g, float& m, float& v) {
  m = __fadd_rn(__fmul_rn(s.beta1, m), __fmul_rn(s.one_minus_beta1, g));
  v = __fadd_rn(__fmul_rn(s.beta2, v), __fmul_rn(s.one_minus_beta2, __fmul_rn(g, g)));
}

// ---- the step ------------------------------------------------------------------------------------
__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One step of two elements, the same bits wherever it is taken: the moments, then the parameter.  Products that
// are added to something are multiply-adds with a -0 that the compiler cannot see: it would contract a packed
// product and a packed sum, which are to be rounded one by one (see opt_moments).  Root and reciprocal are
// approximate, 2 u each: they only reach the parameter.
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

__device__ __forceinline__ void moments_pair(const OptScalars& s, float clip, float2 g, float2& m, float2& v) {
  const float2 zero = both(s.minus_zero);
  g = mul2(g, both(clip));
  m = add2(fma2(both(s.beta1), m, zero), fma2(both(s.one_minus_beta1), g, zero));
  v = add2(fma2(both(s.beta2), v, zero), fma2(both(s.one_minus_beta2), mul2(g, g), zero));
}

__device__ __forceinline__ float2 param_pair(const OptScalars& s, const OptCoefs& c, float2 p, float2 m, float2 v) {
  const float2 d = fma2(make_float2(sqrt_approx(v.x), sqrt_approx(v.y)), both(c.root), both(s.eps));
  return fma2(both(-c.rate), mul2(m, make_float2(rcp_approx(d.x), rcp_approx(d.y))), mul2(p, both(c.decay)));
}

// The approximate root takes subnormal second moments as zero: roots below 2^-63, which with b2 = 0.999 are
// at most 2^-58 in the denominator and nothing beside an eps from here on.  Below it the step is taken with
// IEEE root and division, one element at a time.
constexpr float kLeastEps = 0x1p-33f;

__device__ __forceinline__ void adamw_eight(const OptScalars& s, const OptCoefs& c, float2* p, const float2* g, float2* m, float2* v) {
  if (s.eps >= kLeastEps) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      moments_pair(s, c.clip, g[j], m[j], v[j]);
      p[j] = param_pair(s, c, p[j], m[j], v[j]);
    }
  } else {
    float *ps = reinterpret_cast<float*>(p), *ms = reinterpret_cast<float*>(m), *vs = reinterpret_cast<float*>(v);
    const float* gs = reinterpret_cast<const float*>(g);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      opt_moments(s, __fmul_rn(gs[j], c.clip), ms[j], vs[j]);
      ps[j] = ps[j] * c.decay - c.rate * (ms[j] / (sqrtf(vs[j]) * c.root + s.eps));
    }
  }
}

// ---- 8-bit states -----------------------------------------------------------------------------------
// A 32-bit integer mixing function: two multiplications between three xor-shifts.  Shifts and factors are those that
// Chris Wellons published in 2018 as the best of a search for such functions of little bias.
__device__ __forceinline__ unsigned opt_mix_rest(unsigned x) {
  x *= 0x7feb352du;
  x = (x ^ (x >> 15)) * 0x846ca68bu;
  return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned opt_mix(unsigned x) { return opt_mix_rest(x ^ (x >> 16)); }

// Key of one tensor in one step; the 32 random bits of elements 2 j and 2 j + 1 are
// mix(low 32 bits of j ^ (key + high bits of j)).
__device__ __forceinline__ unsigned opt_key(unsigned seed, unsigned long long t, int index) {
  return opt_mix(opt_mix(opt_mix((unsigned)t) + (unsigned)index) + seed);
}

// ---- host side ---------------------------------------------------------------------------------------
inline size_t opt_size(int dt) { return dt == FLEXSAE_F32 ? 4 : 2; }
inline bool opt_dtype(int dt) { return dt == FLEXSAE_F32 || dt == FLEXSAE_BF16 || dt == FLEXSAE_F16; }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kOptSms = 148;

inline OptTensor make_tensor(const flexsae_optim_tensor& t, int64_t i, int state_bits) {
  OptTensor d;
  d.param = t.param;
  d.grad = t.grad;
  d.exp_avg = t.exp_avg;
  d.exp_avg_sq = t.exp_avg_sq;
  d.exp_avg_scale = t.exp_avg_scale;
  d.exp_avg_sq_scale = t.exp_avg_sq_scale;
  d.master = t.master;
  d.numel = t.numel;
  d.index = (int)i;
  const size_t state = state_bits == 8 ? 8 : 32;
  d.vec = aligned(t.param, 8 * opt_size(t.param_dtype)) && aligned(t.grad, 8 * opt_size(t.grad_dtype)) && aligned(t.master, 32) &&
          aligned(t.exp_avg, state) && aligned(t.exp_avg_sq, state);
  return d;
}

// Kernels are compiled per (parameter type, gradient type, master copy): 0 fp32; then bf16 and fp16,
// each with gradients of its own type or fp32, without and with a master copy.
constexpr int kOptKinds = 9;
inline int kind_of(const flexsae_optim_tensor& t) {
  if (t.param_dtype == FLEXSAE_F32) return 0;
  return 1 + (t.param_dtype == FLEXSAE_F16 ? 4 : 0) + (t.grad_dtype == FLEXSAE_F32 ? 2 : 0) + (t.master ? 1 : 0);
}

// CTAs of `threads` that the GPU holds at the same time, at most `most` per SM: the grid of a launch whose CTAs take
// every gridDim-th chunk, so that all of them run from the start and finish together.  Asked for once (`known`).
template <typename K>
inline cudaError_t resident_ctas(std::atomic<unsigned>& known, K kernel, int threads, int most, unsigned* ctas) {
  *ctas = known.load(std::memory_order_relaxed);
  if (*ctas) return cudaSuccess;
  int n = 0;
  if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0)) return e;
  *ctas = (unsigned)(std::max(1, std::min(n, most)) * kOptSms);
  known.store(*ctas, std::memory_order_relaxed);
  return cudaSuccess;
}

// A launch that is set up while the kernel before it in the stream finishes; every kernel launched so waits for that
// one (opt_wait) before it touches memory.  4096 unit rows of 256 take 5.5 instead of 8.2 us in a row of such
// steps, a model of 20 ragged tensors 43.7 instead of 46.  Letting the next kernel in any earlier (from the start of
// this one) costs more than it gains: 6.4 and 45.4 us.
template <typename Args>
inline cudaError_t launch_early(void (*kernel)(Args), unsigned grid, int threads, const Args& args, cudaStream_t st) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(threads);
  config.stream = st;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args);
}

#define FLEXSAE_OPT_KINDS(kind, CALL)                         \
  switch (kind) {                                             \
    case 0: CALL(float, float, false); break;                 \
    case 1: CALL(__nv_bfloat16, __nv_bfloat16, false); break; \
    case 2: CALL(__nv_bfloat16, __nv_bfloat16, true); break;  \
    case 3: CALL(__nv_bfloat16, float, false); break;         \
    case 4: CALL(__nv_bfloat16, float, true); break;          \
    case 5: CALL(__half, __half, false); break;               \
    case 6: CALL(__half, __half, true); break;                \
    case 7: CALL(__half, float, false); break;                \
    default: CALL(__half, float, true); break;                \
  }

// flexsae_optim_rows.cu: one tensor's unit-row step; `a.cols` and `a.rows` are set.
struct RowArgs {
  OptScalars s;
  OptTensor t;
  long long rows;
  int cols;
  int team;      // threads of a row: 1, 2, ... 32, or the CTA (a multiple of 32)
};
cudaError_t launch_rows(RowArgs a, int kind, cudaStream_t st);

}  // namespace flexsae
