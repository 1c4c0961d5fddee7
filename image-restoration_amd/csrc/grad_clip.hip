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
//
// Bound by memory: the gradients are read twice and written once (the second reading starts with what the cache still
// holds).  Measured a call: 282 fp32 tensors of 26.3 M values into a flat buffer 54 us (316 MB, 5.8 TB/s; the copy of a
// large buffer reaches 4.8), 401 tensors of three types and 60 M values to fp32 107 us, 536 M bf16 593 us (3.2 GB,
// 5.4 TB/s); 24 tensors of 40 k values 7.4 us in one launch (two launches: 12.4).
#include <algorithm>
#include <cmath>
#include <memory>
#include <type_traits>
#include <vector>

#include "runtime.h"

namespace jirf {
namespace {

constexpr int CLIP_T = 256;            // threads that share a chunk
constexpr int CLIP_E = 8;              // elements of a thread's group
constexpr int CLIP_U = 2;              // groups of CLIP_E elements a thread has in flight
constexpr int CLIP_MAX_BLOCKS = 2048;  // eight workgroups per CU
enum { TY_F32 = 0, TY_BF16 = 1, TY_F16 = 2 };

struct ClipChunk {
  const void* src;
  void* dst;              // null: norm only
  unsigned n;             // elements
  unsigned types;         // source type | destination type << 8
};

// Accesses of 8 and 16 bytes at the alignment of one element: the memory instructions take any 2- or 4-byte address.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

// A chunk's addresses come out of memory: said to be device memory here, or every access would take the slower flat path.
template <typename P>
__device__ __forceinline__ const __attribute__((address_space(1))) P* dev(const void* p, size_t byte) {
  return reinterpret_cast<const __attribute__((address_space(1))) P*>(reinterpret_cast<uintptr_t>(p) + byte);
}
template <typename P>
__device__ __forceinline__ __attribute__((address_space(1))) P* dev(void* p, size_t byte) {
  return reinterpret_cast<__attribute__((address_space(1))) P*>(reinterpret_cast<uintptr_t>(p) + byte);
}

// E consecutive elements (4 or 8) as loaded - 8 or 16 bytes, two accesses for eight of fp32 - and as fp32 values.
template <unsigned E> struct Few {
  float f[E];
};
template <int TY, unsigned E> struct FewRaw {
  static constexpr unsigned WORDS = TY == TY_F32 ? E : E / 2;
  unsigned w[WORDS];
  __device__ __forceinline__ void load(const void* p, unsigned g) {
    if constexpr (WORDS == 2) {
      const u32x2 v = *dev<u32x2_a2>(p, g * 8u);
      w[0] = v[0];
      w[1] = v[1];
    } else {
#pragma unroll
      for (unsigned q = 0; q < WORDS / 4; ++q) {
        const u32x4 v = *dev<u32x4_a2>(p, g * (WORDS * 4u) + q * 16u);
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) w[q * 4 + i] = v[i];
      }
    }
  }
  __device__ __forceinline__ Few<E> widen() const {
    Few<E> r;
#pragma unroll
    for (unsigned i = 0; i < E; ++i) {
      if constexpr (TY == TY_F32) r.f[i] = __uint_as_float(w[i]);
      else if constexpr (TY == TY_BF16) r.f[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      else r.f[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
    }
    return r;
  }
};
// A factor outside the normal range of 32 bits (a norm of 1e38 with max_norm 0.01, a grad_scale of 1e60): a factor of order
// one and a power of two on the side where the product stays in range.  (Multiplying in 64 bits instead takes 100 registers
// for 38 in clip_kernel, and spills 241 in norm_clip_kernel.)
struct FarFactor {
  float m;
  int before, after;      // exponents; one of them is 0
};
__device__ __forceinline__ FarFactor far_factor(double k) {
  int e;
  const double f = frexp(k, &e);                                      // [1/2, 1)
  return k < 1.0 ? FarFactor{(float)f, 0, e} : FarFactor{(float)(2.0 * f), e - 1, 0};
}
__device__ __forceinline__ float scaled(float g, float k) { return g * k; }
__device__ __forceinline__ float scaled(float g, const FarFactor& k) {
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(g, k.before) * k.m, k.after);
}
__device__ __forceinline__ bool is_one(float k) { return k == 1.0f; }
__device__ __forceinline__ bool is_one(const FarFactor&) { return false; }
// rounded to nearest even; NT: not kept in the caches
template <typename V, bool NT, typename U>
__device__ __forceinline__ void clip_put(void* p, unsigned byte, U v) {
  if (NT) __builtin_nontemporal_store((V)v, dev<V>(p, byte));
  else *dev<V>(p, byte) = v;
}
template <int TY, unsigned E, bool NT, typename K>
__device__ __forceinline__ void few_store(void* p, unsigned g, const Few<E>& v, K k) {
  constexpr unsigned WORDS = TY == TY_F32 ? E : E / 2;
  unsigned w[WORDS];
#pragma unroll
  for (unsigned i = 0; i < WORDS; ++i) {
    if constexpr (TY == TY_F32) {
      w[i] = __float_as_uint(scaled(v.f[i], k));
    } else {
      typedef typename std::conditional<TY == TY_BF16, __bf16, _Float16>::type H;
      typedef H H2 __attribute__((ext_vector_type(2)));
      H2 h;
      h[0] = (H)scaled(v.f[2 * i], k);
      h[1] = (H)scaled(v.f[2 * i + 1], k);
      w[i] = __builtin_bit_cast(unsigned, h);
    }
  }
  if constexpr (WORDS == 2) {
    clip_put<u32x2_a2, NT>(p, g * 8u, u32x2{w[0], w[1]});
  } else {
#pragma unroll
    for (unsigned q = 0; q < WORDS / 4; ++q)
      clip_put<u32x4_a2, NT>(p, g * (WORDS * 4u) + q * 16u, u32x4{w[q * 4], w[q * 4 + 1], w[q * 4 + 2], w[q * 4 + 3]});
  }
}
template <int TY>
__device__ __forceinline__ float clip_load1(const void* p, unsigned i) {
  if constexpr (TY == TY_F32) return *dev<float>(p, i * 4u);
  else if constexpr (TY == TY_BF16) return __uint_as_float((unsigned)*dev<uint16_t>(p, i * 2u) << 16);
  else return (float)*dev<_Float16>(p, i * 2u);
}
template <int TY>
__device__ __forceinline__ void clip_store1(void* p, unsigned i, float v) {
  if constexpr (TY == TY_F32) *dev<float>(p, i * 4u) = v;
  else if constexpr (TY == TY_BF16) *dev<__bf16>(p, i * 2u) = (__bf16)v;
  else *dev<_Float16>(p, i * 2u) = (_Float16)v;
}
// A maximum that a NaN wins: the bit patterns of |v| order like the values, with every NaN above infinity.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct ClipAcc {
  double sum = 0.0;
  unsigned mx = 0;
};

// One chunk's share of thread `t` of CLIP_T: 16-byte loads at consecutive addresses along the lanes, several in flight.
template <bool MAX, int TY>
__device__ __forceinline__ void norm_chunk(const ClipChunk& ck, unsigned t, ClipAcc& acc) {
  constexpr unsigned E = TY == TY_F32 ? 4 : 8, U = CLIP_U * CLIP_E / E;
  const unsigned groups = ck.n / E;
  auto add = [&](const Few<E>& v) {
#pragma unroll
    for (unsigned i = 0; i < E; ++i) {
      if (MAX) acc.mx = max(acc.mx, abs_bits(v.f[i]));
      else acc.sum = fma((double)v.f[i], (double)v.f[i], acc.sum);
    }
  };
  unsigned g = t;
  for (; g + (U - 1) * CLIP_T < groups; g += U * CLIP_T) {
    FewRaw<TY, E> r[U];
#pragma unroll
    for (unsigned u = 0; u < U; ++u) r[u].load(ck.src, g + u * CLIP_T);
#pragma unroll
    for (unsigned u = 0; u < U; ++u) add(r[u].widen());
  }
  for (; g < groups; g += CLIP_T) {
    FewRaw<TY, E> r;
    r.load(ck.src, g);
    add(r.widen());
  }
  const unsigned i = groups * E + t;
  if (i < ck.n) {
    const float v = clip_load1<TY>(ck.src, i);
    if (MAX) acc.mx = max(acc.mx, abs_bits(v));
    else acc.sum = fma((double)v, (double)v, acc.sum);
  }
}
template <bool MAX>
__device__ __forceinline__ void norm_any(const ClipChunk& ck, unsigned t, ClipAcc& acc) {
  const unsigned ty = ck.types & 0xff;
  if (ty == TY_F32) norm_chunk<MAX, TY_F32>(ck, t, acc);
  else if (ty == TY_BF16) norm_chunk<MAX, TY_BF16>(ck, t, acc);
  else norm_chunk<MAX, TY_F16>(ck, t, acc);
}

// Stores of a wave cover whole 128-byte lines: the elements before the destination's first line and after its last group
// go one by one (a destination packed tight between others starts anywhere; written across lines and past the cache, 105 MB
// became 142 MB of memory traffic).
template <bool NT, int TS, int TD, typename K>
__device__ __forceinline__ void scale_chunk(const ClipChunk& ck, unsigned t, K k) {
  constexpr unsigned E = TS == TY_F32 || TD == TY_F32 ? 4 : 8, U = CLIP_U * CLIP_E / E;
  constexpr unsigned SS = TS == TY_F32 ? 4 : 2, SD = TD == TY_F32 ? 4 : 2;
  const unsigned head = min(ck.n, (128u - ((unsigned)reinterpret_cast<uintptr_t>(ck.dst) & 127u)) % 128u / SD);
  const unsigned groups = (ck.n - head) / E, i = head + groups * E + t;
  const void* src = static_cast<const char*>(ck.src) + head * SS;
  void* dst = static_cast<char*>(ck.dst) + head * SD;
  if (t < head) clip_store1<TD>(ck.dst, t, scaled(clip_load1<TS>(ck.src, t), k));
  unsigned g = t;
  for (; g + (U - 1) * CLIP_T < groups; g += U * CLIP_T) {
    FewRaw<TS, E> r[U];
#pragma unroll
    for (unsigned u = 0; u < U; ++u) r[u].load(src, g + u * CLIP_T);
#pragma unroll
    for (unsigned u = 0; u < U; ++u) few_store<TD, E, NT>(dst, g + u * CLIP_T, r[u].widen(), k);
  }
  for (; g < groups; g += CLIP_T) {
    FewRaw<TS, E> r;
    r.load(src, g);
    few_store<TD, E, NT>(dst, g, r.widen(), k);
  }
  if (i < ck.n) clip_store1<TD>(ck.dst, i, scaled(clip_load1<TS>(ck.src, i), k));
}
template <bool NT, int TS, typename K>
__device__ __forceinline__ void scale_to(const ClipChunk& ck, unsigned t, K k) {
  const unsigned td = ck.types >> 8;
  if (td == TY_F32) scale_chunk<NT, TS, TY_F32>(ck, t, k);
  else if (td == TY_BF16) scale_chunk<NT, TS, TY_BF16>(ck, t, k);
  else scale_chunk<NT, TS, TY_F16>(ck, t, k);
}
template <bool NT, typename K>
__device__ __forceinline__ void scale_any(const ClipChunk& ck, unsigned t, K k) {
  const unsigned ts = ck.types & 0xff;
  // in place with factor 1 every value stays as it is
  if (is_one(k) && ck.src == ck.dst && ts == ck.types >> 8) return;
  if (ts == TY_F32) scale_to<NT, TY_F32>(ck, t, k);
  else if (ts == TY_BF16) scale_to<NT, TY_BF16>(ck, t, k);
  else scale_to<NT, TY_F16>(ck, t, k);
}

// Combines over the workgroup (butterfly in each wave, then the waves in order); the result in every thread.
template <bool MAX>
__device__ __forceinline__ double combine2(double a, double b) {
  if (MAX) return (b > a || b != b) ? b : a;
  return a + b;
}
template <bool MAX, int T>
__device__ __forceinline__ double block_combine(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = combine2<MAX>(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = red[0];
#pragma unroll
  for (int w = 1; w < T / 64; ++w) r = combine2<MAX>(r, red[w]);
  return r;
}

template <bool MAX>
__device__ __forceinline__ double clip_factor(double raw, double max_norm, double grad_scale, double* stats, bool write) {
  const double total = grad_scale * (MAX ? raw : sqrt(raw));
  double k = grad_scale;
  if (max_norm > 0.0) {
    const double c = max_norm / (total + 1e-6);
    k *= c >= 1.0 ? 1.0 : c;           // a NaN norm gives NaN, as the formula does
  }
  if (write) {
    stats[0] = raw;
    stats[1] = total;
    stats[2] = k;
  }
  return k;
}
// Whether 32 bits hold the factor to 24 digits (0 and NaN as they are).
__device__ __forceinline__ bool fits32(double k) { return k == 0.0 || k != k || (k >= 0x1p-126 && k < 0x1p127); }

template <bool MAX>
__global__ __launch_bounds__(CLIP_T) void norm_kernel(const ClipChunk* __restrict__ chunks, int n_chunks,
                                                      double* __restrict__ part) {
  __shared__ double red[CLIP_T / 64];
  ClipAcc acc;
  ClipChunk next = chunks[blockIdx.x];     // (a list with a workgroup has a chunk for it)
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const ClipChunk ck = next;
    if (c + (int)gridDim.x < n_chunks) next = chunks[c + gridDim.x];
    norm_any<MAX>(ck, threadIdx.x, acc);
  }
  const double r = block_combine<MAX, CLIP_T>(MAX ? (double)__uint_as_float(acc.mx) : acc.sum, red);
  if (threadIdx.x == 0) part[blockIdx.x] = r;
}

// The chunks are taken from the last to the first: what norm_kernel read last is what the cache still holds.
template <bool MAX, bool NT>
__global__ __launch_bounds__(CLIP_T) void clip_kernel(const ClipChunk* __restrict__ chunks, int n_chunks,
                                                      const double* __restrict__ part, int n_part, double max_norm,
                                                      double grad_scale, double* __restrict__ stats) {
  __shared__ double red[CLIP_T / 64];
  double t = 0.0;
  for (int i = threadIdx.x; i < n_part; i += CLIP_T) t = combine2<MAX>(t, part[i]);
  const double raw = block_combine<MAX, CLIP_T>(t, red);
  const double k = clip_factor<MAX>(raw, max_norm, grad_scale, stats, blockIdx.x == 0 && threadIdx.x == 0);
  if (fits32(k)) {
    for (int c = n_chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) scale_any<NT>(chunks[c], threadIdx.x, (float)k);
  } else {
    const FarFactor far = far_factor(k);
    for (int c = n_chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) scale_any<NT>(chunks[c], threadIdx.x, far);
  }
}

// Short lists (at most CLIP_SMALL_CHUNKS chunks of CLIP_SMALL_CHUNK elements): one workgroup, one launch.  Teams of two waves
// hold up to eight chunks each in registers between the norm and the store, so memory is waited for once.
constexpr int CLIP_SMALL_T = 128, CLIP_SMALL_TEAMS = 8, CLIP_SMALL_U = 8;
constexpr int CLIP_SMALL_CHUNK = CLIP_SMALL_T * CLIP_E, CLIP_SMALL_CHUNKS = CLIP_SMALL_TEAMS * CLIP_SMALL_U;
template <bool MAX>
__global__ __launch_bounds__(CLIP_SMALL_T * CLIP_SMALL_TEAMS) void norm_clip_kernel(const ClipChunk* __restrict__ chunks, int n_chunks,
                                                                                    int writes, double max_norm, double grad_scale,
                                                                                    double* __restrict__ stats) {
  __shared__ double red[CLIP_SMALL_T * CLIP_SMALL_TEAMS / 64];
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / CLIP_SMALL_T);     // (whole waves)
  const unsigned t = threadIdx.x % CLIP_SMALL_T;
  ClipChunk ck[CLIP_SMALL_U];
#pragma unroll
  for (int u = 0; u < CLIP_SMALL_U; ++u) {
    ck[u] = chunks[min(team + u * CLIP_SMALL_TEAMS, n_chunks - 1)];
    if (team + u * CLIP_SMALL_TEAMS >= n_chunks) ck[u].n = 0;
  }
  // groups of eight, and the few elements past the last whole group; every load is issued before the first is used
  FewRaw<TY_F32, 8> word[CLIP_SMALL_U];         // (16-bit types fill the first half)
  unsigned rt[CLIP_SMALL_U];
#pragma unroll
  for (int u = 0; u < CLIP_SMALL_U; ++u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) word[u].w[i] = 0u;
    rt[u] = 0u;
    const bool wide = (ck[u].types & 0xff) == TY_F32;
    const unsigned groups = ck[u].n / CLIP_E, i = groups * CLIP_E + t;
    if (t < groups) {
      if (wide) {
        word[u].load(ck[u].src, t);
      } else {
        FewRaw<TY_BF16, 8> h;
        h.load(ck[u].src, t);
#pragma unroll
        for (int q = 0; q < 4; ++q) word[u].w[q] = h.w[q];
      }
    }
    if (i < ck[u].n) {
      if (wide) rt[u] = *dev<unsigned>(ck[u].src, i * 4u);
      else rt[u] = *dev<uint16_t>(ck[u].src, i * 2u);
    }
  }
  Few<8> v[CLIP_SMALL_U];
  float tail[CLIP_SMALL_U];
#pragma unroll
  for (int u = 0; u < CLIP_SMALL_U; ++u) {
    const unsigned ty = ck[u].types & 0xff;
    if (ty == TY_F32) {
      v[u] = word[u].widen();
      tail[u] = __uint_as_float(rt[u]);
    } else if (ty == TY_BF16) {
      FewRaw<TY_BF16, 8> h;
#pragma unroll
      for (int q = 0; q < 4; ++q) h.w[q] = word[u].w[q];
      v[u] = h.widen();
      tail[u] = __uint_as_float(rt[u] << 16);
    } else {
      FewRaw<TY_F16, 8> h;
#pragma unroll
      for (int q = 0; q < 4; ++q) h.w[q] = word[u].w[q];
      v[u] = h.widen();
      tail[u] = (float)__builtin_bit_cast(_Float16, (uint16_t)rt[u]);
    }
  }
  ClipAcc acc;
#pragma unroll
  for (int u = 0; u < CLIP_SMALL_U; ++u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (MAX) acc.mx = max(acc.mx, abs_bits(v[u].f[i]));
      else acc.sum = fma((double)v[u].f[i], (double)v[u].f[i], acc.sum);
    }
    if (MAX) acc.mx = max(acc.mx, abs_bits(tail[u]));
    else acc.sum = fma((double)tail[u], (double)tail[u], acc.sum);
  }
  const double raw =
      block_combine<MAX, CLIP_SMALL_T * CLIP_SMALL_TEAMS>(MAX ? (double)__uint_as_float(acc.mx) : acc.sum, red);
  const double kd = clip_factor<MAX>(raw, max_norm, grad_scale, stats, threadIdx.x == 0);
  if (!writes) return;
  float k = (float)kd;
  if (!fits32(kd)) {
    k = 1.0f;
    const FarFactor far = far_factor(kd);
#pragma unroll
    for (int u = 0; u < CLIP_SMALL_U; ++u) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u].f[i] = scaled(v[u].f[i], far);
      tail[u] = scaled(tail[u], far);
    }
  }
#pragma unroll
  for (int u = 0; u < CLIP_SMALL_U; ++u) {
    const unsigned td = ck[u].types >> 8, groups = ck[u].n / CLIP_E, i = groups * CLIP_E + t;
    if (t < groups) {
      if (td == TY_F32) few_store<TY_F32, 8, false>(ck[u].dst, t, v[u], k);
      else if (td == TY_BF16) few_store<TY_BF16, 8, false>(ck[u].dst, t, v[u], k);
      else few_store<TY_F16, 8, false>(ck[u].dst, t, v[u], k);
    }
    if (i < ck[u].n) {
      if (td == TY_F32) clip_store1<TY_F32>(ck[u].dst, i, tail[u] * k);
      else if (td == TY_BF16) clip_store1<TY_BF16>(ck[u].dst, i, tail[u] * k);
      else clip_store1<TY_F16>(ck[u].dst, i, tail[u] * k);
    }
  }
}

struct ClipPlan {
  int device = 0;
  int n_chunks = 0, blocks = 1;
  bool writes = false, small = false;
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
  // in the order of their starts, each range against the earlier ones that have not ended before it starts
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
    // one workgroup takes a small list whole
    long small_chunks = 0;
    for (int i = 0; i < n && small_chunks <= CLIP_SMALL_CHUNKS; ++i) small_chunks += (count[i] + CLIP_SMALL_CHUNK - 1) / CLIP_SMALL_CHUNK;
    plan->small = small_chunks <= CLIP_SMALL_CHUNKS;
    // else about four chunks for every workgroup, of whole steps of CLIP_U groups a thread (4 Ki elements), at most 64 Ki
    const long step = CLIP_T * CLIP_E * CLIP_U;
    const long chunk = plan->small ? CLIP_SMALL_CHUNK
                                   : std::min<long>(65536, std::max<long>(step, (total / (4 * CLIP_MAX_BLOCKS) + step - 1) / step * step));
    long n_chunks = 0;
    for (int i = 0; i < n; ++i) n_chunks += (count[i] + chunk - 1) / chunk;
    JIRF_REQUIRE(n_chunks < 1l << 26, JIRF_EINVAL, "grad_clip_plan_create: too many elements");
    std::vector<ClipChunk> chunks;
    chunks.reserve(std::max(1l, n_chunks));
    for (int i = 0; i < n; ++i) {
      const int ts = type_of(src_dtype[i]), td = dst ? type_of(dst_dtype[i]) : TY_F32;
      for (long o = 0; o < count[i]; o += chunk)
        chunks.push_back({static_cast<const char*>(src[i]) + o * type_bytes(ts),
                          dst ? static_cast<char*>(dst[i]) + o * type_bytes(td) : nullptr,
                          (unsigned)std::min<long>(chunk, count[i] - o), (unsigned)(ts | td << 8)});
      plan->bytes_read += (double)count[i] * type_bytes(ts);
      if (dst) plan->bytes_written += (double)count[i] * type_bytes(td);
    }
    if (chunks.empty()) chunks.push_back({nullptr, nullptr, 0, 0});      // nothing to read, but a row for the kernel
    JIRF_HIP_CHECK(hipGetDevice(&plan->device));
    plan->total = total;
    plan->writes = dst != nullptr;
    plan->n_chunks = (int)chunks.size();
    // the same number of chunks for every workgroup, but the last few
    const int rounds = std::max(1, (plan->n_chunks + CLIP_MAX_BLOCKS - 1) / CLIP_MAX_BLOCKS);
    plan->blocks = std::max(1, (plan->n_chunks + rounds - 1) / rounds);
    plan->chunks.ensure(chunks.size() * sizeof(ClipChunk));
    JIRF_HIP_CHECK(hipMemcpy(plan->chunks.p, chunks.data(), chunks.size() * sizeof(ClipChunk), hipMemcpyHostToDevice));
    *plan_out = plan.release();
    return JIRF_OK;
  });
}

long jirf_train_grad_clip_work_doubles(const void* plan) {
  if (!plan) return -1;
  const ClipPlan* pl = static_cast<const ClipPlan*>(plan);
  return pl->small ? 0 : pl->blocks;
}

int jirf_train_grad_clip_run(const void* plan, int norm_kind, double max_norm, double grad_scale, double* stats, double* work,
                             void* stream) {
  return guarded_c([&] {
    JIRF_REQUIRE(plan && stats && (work || static_cast<const ClipPlan*>(plan)->small), JIRF_EINVAL, "grad_clip_run: null argument");
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
    if (pl->small) {
      Scope sc("train_grad_norm_clip", 3.0 * pl->total, pl->bytes_read + pl->bytes_written, s);
      hipLaunchKernelGGL(mx ? norm_clip_kernel<true> : norm_clip_kernel<false>, dim3(1), dim3(CLIP_SMALL_T * CLIP_SMALL_TEAMS), 0, s, ck, pl->n_chunks,
                         pl->writes ? 1 : 0, max_norm, grad_scale, stats);
      JIRF_HIP_CHECK(hipGetLastError());
      return JIRF_OK;
    }
    {
      Scope sc("train_grad_norm", 2.0 * pl->total, pl->bytes_read, s);
      hipLaunchKernelGGL(mx ? norm_kernel<true> : norm_kernel<false>, dim3(pl->blocks), dim3(CLIP_T), 0, s, ck, pl->n_chunks, work);
    }
    {
      Scope sc("train_grad_clip", 1.0 * pl->total, pl->writes ? pl->bytes_read + pl->bytes_written : 0.0, s);
      // Past half of the 256 MB cache the stores go around it, to leave it to the gradients read a second time (26.3 M
      // fp32 values 67.9 -> 64.5 us, 536 M bf16 661 -> 645 us, both before whole-line stores).
      const bool nt = pl->bytes_read + pl->bytes_written > (128 << 20);
      const auto kernel = mx ? (nt ? clip_kernel<true, true> : clip_kernel<true, false>)
                             : (nt ? clip_kernel<false, true> : clip_kernel<false, false>);
      hipLaunchKernelGGL(kernel, dim3(pl->writes ? pl->blocks : 1), dim3(CLIP_T), 0, s, ck, pl->writes ? pl->n_chunks : 0, work,
                         pl->blocks, max_norm, grad_scale, stats);
    }
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

void jirf_train_grad_clip_plan_destroy(void* plan) { delete static_cast<ClipPlan*>(plan); }

}  // extern "C"
