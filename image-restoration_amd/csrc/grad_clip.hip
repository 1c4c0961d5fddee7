// The global gradient norm over many tensors, and clipping by it (Optimizer.clip_grad_norm,
// basicsr/models/image_restoration_model.py:269-270, whose framework keeps one tensor per parameter).
// jirf_train_sumsq + jirf_train_adam_step do this for one flat fp32 buffer; here the gradients are any number of
// separate fp32 / bf16 / fp16 tensors, and the clipped gradients go back in place or into other memory (the flat
// buffer that the all-reduce and the Adam step take).
//
//   total = grad_scale * sqrt(sum g^2)   or   grad_scale * max |g|
//   k     = grad_scale * min(max_norm / (total + 1e-6), 1)        (max_norm <= 0: k = grad_scale)
//   dst   = k g
//
// Two launches, because no value may be written before the last one has been read: norm_kernel leaves one partial
// result per workgroup, clip_kernel adds them up in every workgroup (the same order everywhere, so all agree to the bit)
// and scales.  Both walk a table of chunks made once per plan: a workgroup takes whole chunks, so tensors of one
// element and of 10^9 share a launch.  Squares and sums are in 64 bits: 32-bit squares overflow at 1.8e19 and a
// 32-bit sum of 10^8 terms loses the small tensors.
#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include "runtime.h"

namespace jirf {
namespace {

constexpr int CLIP_T = 256;            // threads per workgroup
constexpr int CLIP_E = 8;              // elements per thread and step
constexpr int CLIP_MAX_BLOCKS = 2048;  // eight workgroups per CU
enum { TY_F32 = 0, TY_BF16 = 1, TY_F16 = 2 };

struct ClipChunk {
  const void* src;
  void* dst;              // null: norm only
  unsigned n;             // elements
  unsigned types;         // source type | destination type << 8
};

__device__ __forceinline__ float clip_load(const void* p, unsigned ty, long i) {
  if (ty == TY_F32) return static_cast<const float*>(p)[i];
  if (ty == TY_BF16) return __uint_as_float((unsigned)static_cast<const uint16_t*>(p)[i] << 16);
  return (float)static_cast<const _Float16*>(p)[i];
}
// round to nearest even, NaN kept quiet
__device__ __forceinline__ uint16_t to_bf16(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
__device__ __forceinline__ void clip_store(void* p, unsigned ty, long i, float v) {
  if (ty == TY_F32) static_cast<float*>(p)[i] = v;
  else if (ty == TY_BF16) static_cast<uint16_t*>(p)[i] = to_bf16(v);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}
// A maximum that a NaN wins: the bit patterns of |v| order like the values, with every NaN above infinity.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <bool MAX>
__device__ __forceinline__ double block_combine(double v, double* red) {
  const int tid = threadIdx.x;
  red[tid] = v;
  __syncthreads();
  for (int s = CLIP_T / 2; s > 0; s >>= 1) {
    if (tid < s) {
      const double o = red[tid + s];
      if (MAX) red[tid] = (o > red[tid] || o != o) ? o : red[tid];
      else red[tid] += o;
    }
    __syncthreads();
  }
  const double r = red[0];
  __syncthreads();
  return r;
}

template <bool MAX>
__global__ __launch_bounds__(CLIP_T) void norm_kernel(const ClipChunk* __restrict__ chunks, int n_chunks,
                                                      double* __restrict__ part) {
  __shared__ double red[CLIP_T];
  double acc = 0.0;
  unsigned mx = 0;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const ClipChunk ck = chunks[c];
    const unsigned ty = ck.types & 0xff;
    for (unsigned i = threadIdx.x; i < ck.n; i += CLIP_T) {
      const float g = clip_load(ck.src, ty, i);
      if (MAX) mx = max(mx, abs_bits(g));
      else acc = fma((double)g, (double)g, acc);
    }
  }
  const double r = block_combine<MAX>(MAX ? (double)__uint_as_float(mx) : acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = r;
}

template <bool MAX>
__global__ __launch_bounds__(CLIP_T) void clip_kernel(const ClipChunk* __restrict__ chunks, int n_chunks,
                                                      const double* __restrict__ part, int n_part, double max_norm,
                                                      double grad_scale, double* __restrict__ stats) {
  __shared__ double red[CLIP_T];
  double t = 0.0;
  for (int i = threadIdx.x; i < n_part; i += CLIP_T) {
    const double o = part[i];
    if (MAX) t = (o > t || o != o) ? o : t;
    else t += o;
  }
  const double raw = block_combine<MAX>(t, red);
  const double total = grad_scale * (MAX ? raw : sqrt(raw));
  double k = grad_scale;
  if (max_norm > 0.0) {
    const double c = max_norm / (total + 1e-6);
    k *= c >= 1.0 ? 1.0 : c;           // a NaN norm gives NaN, as the formula does
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    stats[0] = raw;
    stats[1] = total;
    stats[2] = k;
  }
  const float kf = (float)k;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const ClipChunk ck = chunks[c];
    if (!ck.dst) continue;
    const unsigned ty = ck.types & 0xff, td = ck.types >> 8;
    for (unsigned i = threadIdx.x; i < ck.n; i += CLIP_T) clip_store(ck.dst, td, i, clip_load(ck.src, ty, i) * kf);
  }
}

struct ClipPlan {
  int device = 0;
  int n_chunks = 0, blocks = 1;
  bool writes = false;
  double bytes_read = 0.0, bytes_written = 0.0;
  long total = 0;
  DeviceBuffer chunks;
};

int type_of(int dtype) { return dtype == JIRF_F32 ? TY_F32 : dtype == JIRF_BF16 ? TY_BF16 : dtype == JIRF_F16 ? TY_F16 : -1; }
int type_bytes(int ty) { return ty == TY_F32 ? 4 : 2; }

template <typename F>
int guarded_c(F&& f) {
  try {
    return f();
  } catch (const Failure& e) {
    return e.code;
  } catch (const std::bad_alloc&) {
    set_error("host allocation failed");
    return JIRF_ENOMEM;
  } catch (...) {
    set_error("unexpected failure");
    return JIRF_EINVAL;
  }
}

// A destination may be its own source (in place) and must not touch any other source or destination: two
// workgroups would write one place, or one would read what another has scaled already.
void check_ranges(int n, const void* const* src, const int* sdt, void* const* dst, const int* ddt, const long* count) {
  struct Range {
    uintptr_t lo, hi;
    int i;
    bool is_dst;
  };
  std::vector<Range> r;
  for (int i = 0; i < n; ++i) {
    if (count[i] == 0) continue;
    const uintptr_t s = reinterpret_cast<uintptr_t>(src[i]), d = reinterpret_cast<uintptr_t>(dst[i]);
    const uintptr_t sb = (uintptr_t)count[i] * type_bytes(type_of(sdt[i]));
    r.push_back({s, s + sb, i, false});
    r.push_back({d, d + (uintptr_t)count[i] * type_bytes(type_of(ddt[i])), i, true});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  // sweep: the furthest end so far of any source and of any destination, and of any by another tensor
  std::vector<const Range*> open;
  for (const Range& a : r) {
    size_t keep = 0;
    for (const Range* o : open)
      if (o->hi > a.lo) open[keep++] = o;
    open.resize(keep);
    for (const Range* o : open) {
      if (!o->is_dst && !a.is_dst) continue;                       // sources may share memory
      const bool in_place = o->i == a.i && o->lo == a.lo && o->hi == a.hi && o->is_dst != a.is_dst;
      JIRF_REQUIRE(in_place, JIRF_EINVAL, "grad_clip: the destination of tensor %d overlaps tensor %d", o->is_dst ? o->i : a.i,
                   o->is_dst ? a.i : o->i);
    }
    open.push_back(&a);
  }
}

}  // namespace
}  // namespace jirf

using namespace jirf;

extern "C" {

int jirf_train_grad_clip_plan_create(int n, const void* const* src, const int* src_dtype, void* const* dst,
                                     const int* dst_dtype, const long* count, void** plan_out) {
  return guarded_c([&] {
    JIRF_REQUIRE(n > 0 && src && src_dtype && count && plan_out && (!dst || dst_dtype), JIRF_EINVAL,
                 "grad_clip_plan_create: bad arguments");
    long total = 0;
    for (int i = 0; i < n; ++i) {
      JIRF_REQUIRE(count[i] >= 0 && (count[i] == 0 || (src[i] && (!dst || dst[i]))), JIRF_EINVAL,
                   "grad_clip_plan_create: tensor %d: null pointer or negative size", i);
      JIRF_REQUIRE(type_of(src_dtype[i]) >= 0 && (!dst || type_of(dst_dtype[i]) >= 0), JIRF_EINVAL,
                   "grad_clip_plan_create: tensor %d: only fp32, bf16 and fp16", i);
      const uintptr_t sm = type_bytes(type_of(src_dtype[i])) - 1, dm = dst ? type_bytes(type_of(dst_dtype[i])) - 1 : 0;
      JIRF_REQUIRE((reinterpret_cast<uintptr_t>(src[i]) & sm) == 0 && (!dst || (reinterpret_cast<uintptr_t>(dst[i]) & dm) == 0),
                   JIRF_EINVAL, "grad_clip_plan_create: tensor %d is not aligned to its elements", i);
      JIRF_REQUIRE(count[i] <= (1l << 46) && total <= (1l << 46), JIRF_EINVAL, "grad_clip_plan_create: tensor %d is too large", i);
      total += count[i];
    }
    if (dst) check_ranges(n, src, src_dtype, dst, dst_dtype, count);
    auto plan = std::make_unique<ClipPlan>();
    // enough chunks to occupy every workgroup, at least one step of a workgroup each, at most 64 Ki elements
    const long step = CLIP_T * CLIP_E;
    const long chunk = std::min<long>(65536, std::max<long>(step, (total / CLIP_MAX_BLOCKS + step - 1) / step * step));
    std::vector<ClipChunk> chunks;
    for (int i = 0; i < n; ++i) {
      const int ts = type_of(src_dtype[i]), td = dst ? type_of(dst_dtype[i]) : TY_F32;
      for (long o = 0; o < count[i]; o += chunk)
        chunks.push_back({static_cast<const char*>(src[i]) + o * type_bytes(ts),
                          dst ? static_cast<char*>(dst[i]) + o * type_bytes(td) : nullptr,
                          (unsigned)std::min<long>(chunk, count[i] - o), (unsigned)(ts | td << 8)});
      plan->bytes_read += (double)count[i] * type_bytes(ts);
      if (dst) plan->bytes_written += (double)count[i] * type_bytes(td);
    }
    JIRF_REQUIRE(chunks.size() < (size_t)1 << 30, JIRF_EINVAL, "grad_clip_plan_create: too many elements");
    JIRF_HIP_CHECK(hipGetDevice(&plan->device));
    plan->total = total;
    plan->writes = dst != nullptr;
    plan->n_chunks = (int)chunks.size();
    plan->blocks = std::max(1, std::min(CLIP_MAX_BLOCKS, plan->n_chunks));
    if (!chunks.empty()) {
      plan->chunks.ensure(chunks.size() * sizeof(ClipChunk));
      JIRF_HIP_CHECK(hipMemcpy(plan->chunks.p, chunks.data(), chunks.size() * sizeof(ClipChunk), hipMemcpyHostToDevice));
    }
    *plan_out = plan.release();
    return JIRF_OK;
  });
}

long jirf_train_grad_clip_work_doubles(const void* plan) {
  return plan ? static_cast<const ClipPlan*>(plan)->blocks : -1;
}

int jirf_train_grad_clip_run(const void* plan, int norm_kind, double max_norm, double grad_scale, double* stats, double* work,
                             void* stream) {
  return guarded_c([&] {
    JIRF_REQUIRE(plan && stats && work, JIRF_EINVAL, "grad_clip_run: null argument");
    JIRF_REQUIRE(norm_kind == JIRF_NORM_L2 || norm_kind == JIRF_NORM_MAX, JIRF_EINVAL, "grad_clip_run: norm_kind %d", norm_kind);
    JIRF_REQUIRE(grad_scale > 0.0 && std::isfinite(grad_scale) && !std::isnan(max_norm), JIRF_EINVAL,
                 "grad_clip_run: grad_scale must be positive and finite, max_norm a number");
    const ClipPlan* pl = static_cast<const ClipPlan*>(plan);
    int dev = 0;
    JIRF_HIP_CHECK(hipGetDevice(&dev));
    JIRF_REQUIRE(dev == pl->device, JIRF_EINVAL, "grad_clip_run: the plan belongs to device %d, current device %d", pl->device, dev);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const ClipChunk* ck = static_cast<const ClipChunk*>(pl->chunks.p);
    const bool mx = norm_kind == JIRF_NORM_MAX;
    {
      Scope sc("train_grad_norm", 2.0 * pl->total, pl->bytes_read, s);
      hipLaunchKernelGGL(mx ? norm_kernel<true> : norm_kernel<false>, dim3(pl->blocks), dim3(CLIP_T), 0, s, ck, pl->n_chunks, work);
    }
    {
      Scope sc("train_grad_clip", 1.0 * pl->total, pl->writes ? pl->bytes_read + pl->bytes_written : 0.0, s);
      hipLaunchKernelGGL(mx ? clip_kernel<true> : clip_kernel<false>, dim3(pl->writes ? pl->blocks : 1), dim3(CLIP_T), 0, s, ck,
                         pl->writes ? pl->n_chunks : 0, work, pl->blocks, max_norm, grad_scale, stats);
    }
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

void jirf_train_grad_clip_plan_destroy(void* plan) { delete static_cast<ClipPlan*>(plan); }

}  // extern "C"
