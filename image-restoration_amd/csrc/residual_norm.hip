// The join of a residual block with the norms on both sides of it, forward and backward:
//
//   u = N_post(f)  (or f)          the branch's output, normalised after the block
//   y = x + scale[b] * gate * u    residual stream; scale = a sample's DropPath factor, gate = a layer scale [C] or a
//                                  modulation [B][C]
//   n = N_pre(y)                   the next branch's input, normalised before the block
//
// (AST's block is x + drop_path(attn(norm1(x))) followed by norm2, ast_arch.py:768-842: scale and N_pre.)  With
// mu = mean_c v, var = mean_c (v - mu)^2 per token (pixel):
//   kind 1  (v - mu) rs w + b,  rs = (var + eps)^-1/2        nn.LayerNorm, hint_arch.py:120-145 "WithBias"
//   kind 2  v rs w,             rs = (var + eps)^-1/2        hint_arch.py:98-117 "BiasFree"
//   kind 3  v rs w,             rs = (mean v^2 + eps)^-1/2   root mean square (mu := 0)
// Backward of one norm, with vh = (v - mu) rs (kind 1) or v rs (2, 3), c = (v - mu) rs and g = dOut w:
//   dv = rs (g - [kind 1] mean_c g - c mean_c(g vh)),   dw = sum dOut vh,   db = sum dOut
// so for the join, with dyt = dy + dN_pre(dn):
//   dx = dyt,   du = scale gate dyt,   dgate = sum scale u dyt,   df = dN_post(du)
//
// Activations fp32, bf16 or fp16, all arithmetic fp32, one rounding per stored value: n is formed from the fp32 sum and
// not from the rounded y, and the statistics saved for the backward are those of the fp32 values.  Parameters, gate, scale,
// statistics and parameter gradients are fp32.  No atomics: every sum has a fixed order.
#include <algorithm>
#include <cmath>

#include "runtime.h"

namespace jirf {
namespace {

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float ld(const float* p) { return *p; }
  static __device__ __forceinline__ void st(float* p, float v) { *p = v; }
};
template <> struct Elem<__bf16> {
  static __device__ __forceinline__ float ld(const __bf16* p) { return (float)*p; }
  static __device__ __forceinline__ void st(__bf16* p, float v) { *p = (__bf16)v; }
};
template <> struct Elem<_Float16> {
  static __device__ __forceinline__ float ld(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ void st(_Float16* p, float v) { *p = (_Float16)v; }
};

struct RnArgs {
  // activations, element (b, c, p) at ptr + b * bs + c * cs + p * ps
  const void *x, *f, *dy, *dn, *y_in;
  void *y, *n, *dx, *df;
  long x_bs, f_bs, dy_bs, dn_bs, yi_bs, y_bs, n_bs, dx_bs, df_bs;
  long cs, ps;
  const float *post_w, *post_b, *gate, *scale, *pre_w, *pre_b;
  const float* stats_in;   // [4][B][P]
  float* stats;            // [4][B][P] or null
  float* rowsum;           // backward: [2][B][P], the two row means of the pre norm's gradient
  float* part;             // backward: [5][workers][C] partial parameter gradients
  float* part_gate;        // backward, gate kind 2 and S > 1: [B][S][C]
  float* dgate;            // backward, gate kind 2 and S == 1: written directly
  int post, pre, gate_kind, accumulate;
  float eps;
  int B, C, P;
  int S, ipw;              // workers per image (ipw == 1), or images per worker (S == 1)
};
enum { Q_POST_W = 0, Q_POST_B = 1, Q_GATE = 2, Q_PRE_W = 3, Q_PRE_B = 4, Q_N = 5 };

// ---- any number of channels -------------------------------------------------------------------------------------------
// One workgroup per token (tokens layout, 256 threads along the channels) or per 64 pixels (planar, four waves along
// the channels); nothing is kept between the passes over the channels, each reads its operands again.
template <bool TOK>
struct Sweep {
  float* red;
  // sum over the threads that share a token
  __device__ __forceinline__ float sum(float v) const {
    const int tid = threadIdx.x;
    __syncthreads();
    if (TOK) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
      if ((tid & 63) == 0) red[tid >> 6] = v;
      __syncthreads();
      return (red[0] + red[1]) + (red[2] + red[3]);
    }
    red[tid] = v;
    __syncthreads();
    const int l = tid & 63;
    return (red[l] + red[64 + l]) + (red[128 + l] + red[192 + l]);
  }
};

template <typename T, bool TOK>
__global__ __launch_bounds__(256) void rn_fwd_sweep(const RnArgs a) {
  __shared__ float red[256];
  const Sweep<TOK> sw{red};
  const int tid = threadIdx.x;
  const long tiles = TOK ? a.P : (a.P + 63) / 64;
  const int c0 = TOK ? tid : tid >> 6, dc = TOK ? 256 : 4;
  const float inv = 1.0f / (float)a.C;
  for (long t = blockIdx.x; t < tiles * a.B; t += gridDim.x) {
    const long b = t / tiles, pt = t % tiles;
    const long p = TOK ? pt : pt * 64 + (tid & 63);
    const bool on = p < a.P;
    const long o = (on ? p : 0) * a.ps;
    const T* x = static_cast<const T*>(a.x) + b * a.x_bs + o;
    const T* f = static_cast<const T*>(a.f) + b * a.f_bs + o;
    T* y = static_cast<T*>(a.y) + b * a.y_bs + o;
    T* n = static_cast<T*>(a.n) + (a.pre ? b * a.n_bs + o : 0);
    const float s = a.scale ? a.scale[b] : 1.0f;
    const float* gate = a.gate_kind == 2 ? a.gate + b * a.C : a.gate;
    float mu0 = 0.f, rs0 = 0.f, mu1 = 0.f, rs1 = 0.f;
    if (a.post) {
      float q = 0.f;
      if (a.post != 3) {
        for (int c = c0; c < a.C; c += dc) q += Elem<T>::ld(f + c * a.cs);
        mu0 = sw.sum(q) * inv;
      }
      q = 0.f;
      for (int c = c0; c < a.C; c += dc) {
        const float d = Elem<T>::ld(f + c * a.cs) - mu0;
        q = fmaf(d, d, q);
      }
      rs0 = 1.0f / sqrtf(sw.sum(q) * inv + a.eps);
    }
    auto join = [&](int c) {
      float u = Elem<T>::ld(f + c * a.cs);
      if (a.post) {
        u = (a.post == 1 ? u - mu0 : u) * rs0 * a.post_w[c];
        if (a.post == 1 && a.post_b) u += a.post_b[c];
      }
      return fmaf(a.gate_kind ? s * gate[c] : s, u, Elem<T>::ld(x + c * a.cs));
    };
    if (a.pre) {
      float q = 0.f;
      if (a.pre != 3) {
        for (int c = c0; c < a.C; c += dc) q += join(c);
        mu1 = sw.sum(q) * inv;
      }
      q = 0.f;
      for (int c = c0; c < a.C; c += dc) {
        const float d = join(c) - mu1;
        q = fmaf(d, d, q);
      }
      rs1 = 1.0f / sqrtf(sw.sum(q) * inv + a.eps);
    }
    if (on) {
      for (int c = c0; c < a.C; c += dc) {      // y may be x and n may be f: a thread reads both before it writes
        const float v = join(c);
        Elem<T>::st(y + c * a.cs, v);
        if (a.pre) {
          float r = (a.pre == 1 ? v - mu1 : v) * rs1 * a.pre_w[c];
          if (a.pre == 1 && a.pre_b) r += a.pre_b[c];
          Elem<T>::st(n + c * a.cs, r);
        }
      }
      if (a.stats && c0 == 0) {
        const long bp = (long)a.B * a.P, at = b * a.P + p;
        a.stats[at] = mu0;
        a.stats[bp + at] = rs0;
        a.stats[2 * bp + at] = mu1;
        a.stats[3 * bp + at] = rs1;
      }
    }
  }
}

// What the backward's element formulas need of one token.
struct RowBwd {
  float mu0, rs0, mu1, rs1, m1, m2, s;
};

// dyt of one element: dy + rs (g - [kind 1] mean g - c mean(g vh))
__device__ __forceinline__ float rn_dyt(const RnArgs& a, const RowBwd& r, float dy, float dn, float y, float w) {
  if (!a.pre) return dy;
  return dy + r.rs1 * (dn * w - r.m1 - (y - r.mu1) * r.rs1 * r.m2);
}

template <typename T, bool TOK>
__global__ __launch_bounds__(256) void rn_bwd_sweep(const RnArgs a) {
  __shared__ float red[256];
  const Sweep<TOK> sw{red};
  const int tid = threadIdx.x;
  const long tiles = TOK ? a.P : (a.P + 63) / 64;
  const int c0 = TOK ? tid : tid >> 6, dc = TOK ? 256 : 4;
  const float inv = 1.0f / (float)a.C;
  const long bp = (long)a.B * a.P;
  for (long t = blockIdx.x; t < tiles * a.B; t += gridDim.x) {
    const long b = t / tiles, pt = t % tiles;
    const long p = TOK ? pt : pt * 64 + (tid & 63);
    const bool on = p < a.P;
    const long o = (on ? p : 0) * a.ps, at = b * a.P + (on ? p : 0);
    const T* dy = a.dy ? static_cast<const T*>(a.dy) + b * a.dy_bs + o : nullptr;
    const T* dn = a.pre ? static_cast<const T*>(a.dn) + b * a.dn_bs + o : nullptr;
    const T* y = a.pre ? static_cast<const T*>(a.y_in) + b * a.yi_bs + o : nullptr;
    const T* f = a.post ? static_cast<const T*>(a.f) + b * a.f_bs + o : nullptr;
    T* dx = static_cast<T*>(a.dx) + b * a.dx_bs + o;
    T* df = static_cast<T*>(a.df) + b * a.df_bs + o;
    const float* gate = a.gate_kind == 2 ? a.gate + b * a.C : a.gate;
    RowBwd r{};
    r.s = a.scale ? a.scale[b] : 1.0f;
    if (a.post) {
      r.mu0 = a.stats_in[at];
      r.rs0 = a.stats_in[bp + at];
    }
    if (a.pre) {
      r.mu1 = a.stats_in[2 * bp + at];
      r.rs1 = a.stats_in[3 * bp + at];
      const float m = a.pre == 1 ? r.mu1 : 0.f;
      float s1 = 0.f, s2 = 0.f;
      for (int c = c0; c < a.C; c += dc) {
        const float g = Elem<T>::ld(dn + c * a.cs) * a.pre_w[c];
        s1 += g;
        s2 = fmaf(g, (Elem<T>::ld(y + c * a.cs) - m) * r.rs1, s2);
      }
      r.m1 = a.pre == 1 ? sw.sum(s1) * inv : 0.f;
      r.m2 = sw.sum(s2) * inv;
      if (on && c0 == 0) {
        a.rowsum[at] = r.m1;
        a.rowsum[bp + at] = r.m2;
      }
    }
    auto dyt = [&](int c) {
      return rn_dyt(a, r, dy ? Elem<T>::ld(dy + c * a.cs) : 0.f, a.pre ? Elem<T>::ld(dn + c * a.cs) : 0.f,
                    a.pre ? Elem<T>::ld(y + c * a.cs) : 0.f, a.pre ? a.pre_w[c] : 0.f);
    };
    float t1 = 0.f, t2 = 0.f;
    if (a.post) {
      const float m = a.post == 1 ? r.mu0 : 0.f;
      for (int c = c0; c < a.C; c += dc) {
        const float g = dyt(c) * (a.gate_kind ? r.s * gate[c] : r.s) * a.post_w[c];
        t1 += g;
        t2 = fmaf(g, (Elem<T>::ld(f + c * a.cs) - m) * r.rs0, t2);
      }
      t1 = a.post == 1 ? sw.sum(t1) * inv : 0.f;
      t2 = sw.sum(t2) * inv;
    }
    if (on)
      for (int c = c0; c < a.C; c += dc) {
        const float d = dyt(c);
        float du = d * (a.gate_kind ? r.s * gate[c] : r.s);
        if (a.post) du = r.rs0 * (du * a.post_w[c] - t1 - (Elem<T>::ld(f + c * a.cs) - r.mu0) * r.rs0 * t2);
        Elem<T>::st(dx + c * a.cs, d);
        Elem<T>::st(df + c * a.cs, du);
      }
  }
}

// The parameter gradients of the sweep form: one pass more over the operands, a workgroup per 64 channels and worker
// (tokens: lanes along the channels, waves along the rows; planar: a wave per channel, lanes along the pixels).
template <typename T, bool TOK>
__global__ __launch_bounds__(256) void rn_bwd_params_sweep(const RnArgs a) {
  __shared__ float red[Q_N][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int worker = blockIdx.y;
  const int b0 = a.S > 1 ? worker / a.S : worker * a.ipw, b1 = min(a.B, a.S > 1 ? b0 + 1 : b0 + a.ipw);
  const int slab = a.S > 1 ? worker % a.S : 0;
  const int per = (a.P + a.S - 1) / a.S, p0 = min(a.P, slab * per), p1 = min(a.P, p0 + per);
  const long bp = (long)a.B * a.P;
  const int c = blockIdx.x * (TOK ? 64 : 4) + (TOK ? lane : wave);
  const bool on = c < a.C;
  const int cc = on ? c : 0;
  float acc[Q_N] = {0.f, 0.f, 0.f, 0.f, 0.f};
  // per-channel sums across the threads that share the channel
  auto total = [&](float v, float* buf) {
    if (!TOK) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
      return v;
    }
    __syncthreads();
    buf[tid] = v;
    __syncthreads();
    return (buf[lane] + buf[64 + lane]) + (buf[128 + lane] + buf[192 + lane]);
  };
  const bool writer = on && (TOK ? wave == 0 : lane == 0);
  for (int b = b0; b < b1; ++b) {
    const float s = a.scale ? a.scale[b] : 1.0f;
    const float gt = a.gate_kind == 2 ? a.gate[(long)b * a.C + cc] : a.gate_kind ? a.gate[cc] : 1.0f;
    const float w1 = a.pre ? a.pre_w[cc] : 0.f, w0 = a.post ? a.post_w[cc] : 1.f;
    const float b0v = a.post == 1 && a.post_b ? a.post_b[cc] : 0.f;
    float gacc = 0.f;
    for (int p = p0 + (TOK ? wave : lane); p < p1; p += TOK ? 4 : 64) {
      const long o = p * a.ps + cc * a.cs, at = (long)b * a.P + p;
      RowBwd r{};
      float dnv = 0.f, yv = 0.f;
      if (a.pre) {
        r.mu1 = a.stats_in[2 * bp + at];
        r.rs1 = a.stats_in[3 * bp + at];
        r.m1 = a.rowsum[at];
        r.m2 = a.rowsum[bp + at];
        dnv = Elem<T>::ld(static_cast<const T*>(a.dn) + b * a.dn_bs + o);
        yv = Elem<T>::ld(static_cast<const T*>(a.y_in) + b * a.yi_bs + o);
        acc[Q_PRE_W] = fmaf(dnv, (a.pre == 1 ? yv - r.mu1 : yv) * r.rs1, acc[Q_PRE_W]);
        acc[Q_PRE_B] += dnv;
      }
      if (!a.post && !a.gate_kind) continue;
      const float d = rn_dyt(a, r, a.dy ? Elem<T>::ld(static_cast<const T*>(a.dy) + b * a.dy_bs + o) : 0.f, dnv, yv, w1) * s;
      float u = Elem<T>::ld(static_cast<const T*>(a.f) + b * a.f_bs + o);
      if (a.post) {
        u = (a.post == 1 ? u - a.stats_in[at] : u) * a.stats_in[bp + at];
        acc[Q_POST_W] = fmaf(d * gt, u, acc[Q_POST_W]);
        acc[Q_POST_B] += d * gt;
        u = fmaf(u, w0, b0v);
      }
      gacc = fmaf(d, u, gacc);
    }
    if (a.gate_kind == 2) {
      const float g = total(gacc, red[Q_GATE]);
      if (writer) {
        if (a.S > 1) a.part_gate[((long)b * a.S + slab) * a.C + c] = g;
        else if (a.dgate) a.dgate[(long)b * a.C + c] = a.accumulate ? a.dgate[(long)b * a.C + c] + g : g;
      }
    } else {
      acc[Q_GATE] += gacc;
    }
  }
  const long workers = gridDim.y;
#pragma unroll
  for (int q = 0; q < Q_N; ++q) {
    const float v = total(acc[q], red[q]);
    if (writer) a.part[((long)q * workers + worker) * a.C + c] = v;
  }
}

// out[g][c] (+)= sum over rows r of part[g][r][c], rows in order per thread, then the row lanes in order, in 64 bits.
// blockIdx.y: quantity; a null out skips it.
struct ReduceArgs {
  const float* part[Q_N];
  float* out[Q_N];
  long rows, C;
  int accumulate;
};
__global__ __launch_bounds__(1024) void rn_reduce(const ReduceArgs a) {
  __shared__ double red[32][33];
  const float* part = a.part[blockIdx.y] + (long)blockIdx.z * a.rows * a.C;
  float* out = a.out[blockIdx.y] + (long)blockIdx.z * a.C;
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const long c = (long)blockIdx.x * 32 + cl;
  double t = 0.0;
  if (c < a.C)
    for (long r = rl; r < a.rows; r += 32) t += (double)part[r * a.C + c];
  red[rl][cl] = t;
  __syncthreads();
  if (rl == 0 && c < a.C) {
    double v = 0.0;
#pragma unroll
    for (int r = 0; r < 32; ++r) v += red[r][cl];
    out[c] = a.accumulate ? (float)((double)out[c] + v) : (float)v;
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------
template <typename F>
int guarded_r(F&& f) {
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

bool kind_ok(int k) { return k >= 0 && k <= 3; }
bool dtype_ok(int d) { return d == JIRF_F32 || d == JIRF_BF16 || d == JIRF_F16; }

void check_common(const char* who, int dtype, int layout, int post, const float* post_w, int gate_kind, const float* gate, int pre,
                  const float* pre_w, int B, int C, int P) {
  JIRF_REQUIRE(dtype_ok(dtype), JIRF_EINVAL, "%s: dtype %d (only fp32, bf16 and fp16)", who, dtype);
  JIRF_REQUIRE(layout == JIRF_LAYOUT_PLANAR || layout == JIRF_LAYOUT_TOKENS, JIRF_EINVAL, "%s: layout %d", who, layout);
  JIRF_REQUIRE(kind_ok(post) && kind_ok(pre) && gate_kind >= 0 && gate_kind <= 2, JIRF_EINVAL,
               "%s: norm kinds are 0..3 and gate kinds 0..2, got post %d, pre %d, gate %d", who, post, pre, gate_kind);
  JIRF_REQUIRE((!post || post_w) && (!pre || pre_w) && (!gate_kind || gate), JIRF_EINVAL,
               "%s: a norm without its weight or a gate without its factors", who);
  JIRF_REQUIRE(B > 0 && C > 0 && P > 0, JIRF_EINVAL, "%s: sizes B %d C %d P %d", who, B, C, P);
}
// Batch stride of one tensor (0: dense).  An image's C * P elements are contiguous; images of an output may not overlap.
long batch_stride(const char* who, const char* name, const void* p, long bs, int dtype, int B, int C, int P) {
  const long n = (long)C * P;
  JIRF_REQUIRE((reinterpret_cast<uintptr_t>(p) & (dtype == JIRF_F32 ? 3 : 1)) == 0, JIRF_EINVAL,
               "%s: %s is not aligned to its elements", who, name);
  JIRF_REQUIRE(bs == 0 || bs >= n || B == 1, JIRF_EINVAL, "%s: batch stride %ld of %s is less than C * P = %ld", who, bs, name, n);
  return bs ? bs : n;
}
// A tensor of the call: B images of n contiguous elements, bs apart.
struct Span {
  const char* name;
  const void* p;
  long bs;
};
// Refuses an output that touches another tensor of the call.  Images of equal stride interleave without touching (channel
// slices of one wider buffer); where the strides differ, overlapping extents are refused.  same_ok: the output may be
// exactly that tensor.
void check_apart(const char* who, const Span& out, const Span& other, int dtype, int B, int C, int P, bool same_ok) {
  if (!out.p || !other.p) return;
  const long es = dtype == JIRF_F32 ? 4 : 2, n = (long)C * P * es, so = out.bs * es, st = other.bs * es;
  const long a = (long)reinterpret_cast<uintptr_t>(out.p), b = (long)reinterpret_cast<uintptr_t>(other.p);
  if (same_ok && a == b && (so == st || B == 1)) return;
  if (a + (B - 1) * so + n <= b || b + (B - 1) * st + n <= a) return;
  bool touch = true;
  if (B > 1 && so == st) {
    const long r = ((b - a) % so + so) % so;
    touch = r < n || r > so - n;
  }
  JIRF_REQUIRE(!touch, JIRF_EINVAL, "%s: %s overlaps %s", who, out.name, other.name);
}
void set_layout(RnArgs& a, int layout) {
  a.cs = layout == JIRF_LAYOUT_TOKENS ? 1 : a.P;
  a.ps = layout == JIRF_LAYOUT_TOKENS ? a.C : 1;
}

#define RN_DISPATCH(dtype, tok, KERNEL, grid, block, s, args)                                                  \
  do {                                                                                                         \
    if (dtype == JIRF_F32) {                                                                                   \
      if (tok) hipLaunchKernelGGL((KERNEL<float, true>), grid, block, 0, s, args);                             \
      else hipLaunchKernelGGL((KERNEL<float, false>), grid, block, 0, s, args);                                \
    } else if (dtype == JIRF_BF16) {                                                                           \
      if (tok) hipLaunchKernelGGL((KERNEL<__bf16, true>), grid, block, 0, s, args);                            \
      else hipLaunchKernelGGL((KERNEL<__bf16, false>), grid, block, 0, s, args);                               \
    } else {                                                                                                   \
      if (tok) hipLaunchKernelGGL((KERNEL<_Float16, true>), grid, block, 0, s, args);                          \
      else hipLaunchKernelGGL((KERNEL<_Float16, false>), grid, block, 0, s, args);                             \
    }                                                                                                          \
  } while (0)

unsigned sweep_grid(bool tok, int B, int P) {
  const long tiles = (tok ? (long)P : ((long)P + 63) / 64) * B;
  return (unsigned)std::min<long>(tiles, 1 << 16);
}

// Workers of the parameter gradients: at least 64 pixels each, about 256 of them.
void bwd_workers(RnArgs& a) {
  const int want = 256;
  if (a.B >= want) {
    a.S = 1;
    a.ipw = (a.B + want - 1) / want;
  } else {
    a.ipw = 1;
    a.S = (int)std::max<long>(1, std::min<long>((a.P + 63) / 64, want / a.B));
  }
}
long n_workers(const RnArgs& a) { return a.S > 1 ? (long)a.B * a.S : ((long)a.B + a.ipw - 1) / a.ipw; }

struct BwdWork {
  long rowsum, part, part_gate, total;   // floats
};
BwdWork bwd_work(const RnArgs& a) {
  BwdWork w{};
  w.rowsum = a.pre ? 2l * a.B * a.P : 0;
  w.part = (long)Q_N * n_workers(a) * a.C;
  w.part_gate = a.gate_kind == 2 && a.S > 1 ? (long)a.B * a.S * a.C : 0;
  w.total = w.rowsum + w.part + w.part_gate;
  return w;
}

}  // namespace
}  // namespace jirf

using namespace jirf;

extern "C" {

int jirf_train_residual_norm(const void* x, long x_bs, const void* f, long f_bs, int dtype, int layout, int post_kind,
                             const float* post_w, const float* post_b, int gate_kind, const float* gate, const float* scale,
                             int pre_kind, const float* pre_w, const float* pre_b, float eps, void* y, long y_bs, void* n,
                             long n_bs, float* stats, int B, int C, int P, void* stream) {
  return guarded_r([&] {
    const char* who = "residual_norm";
    check_common(who, dtype, layout, post_kind, post_w, gate_kind, gate, pre_kind, pre_w, B, C, P);
    JIRF_REQUIRE(x && f && y && (!pre_kind || n), JIRF_EINVAL, "%s: null activation", who);
    JIRF_REQUIRE(eps >= 0.f && std::isfinite(eps), JIRF_EINVAL, "%s: eps must be finite and not negative", who);
    RnArgs a{};
    a.x = x; a.f = f; a.y = y; a.n = n;
    a.x_bs = batch_stride(who, "x", x, x_bs, dtype, B, C, P);
    a.f_bs = batch_stride(who, "f", f, f_bs, dtype, B, C, P);
    a.y_bs = batch_stride(who, "y", y, y_bs, dtype, B, C, P);
    a.n_bs = pre_kind ? batch_stride(who, "n", n, n_bs, dtype, B, C, P) : 0;
    const Span sx{"x", x, a.x_bs}, sf{"f", f, a.f_bs}, sy{"y", y, a.y_bs}, sn{"n", pre_kind ? n : nullptr, a.n_bs};
    check_apart(who, sy, sx, dtype, B, C, P, true);
    check_apart(who, sy, sf, dtype, B, C, P, false);
    check_apart(who, sn, sx, dtype, B, C, P, false);
    check_apart(who, sn, sf, dtype, B, C, P, true);
    check_apart(who, sn, sy, dtype, B, C, P, false);
    a.post = post_kind; a.pre = pre_kind; a.gate_kind = gate_kind;
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b; a.gate = gate; a.scale = scale;
    a.eps = eps; a.stats = stats; a.B = B; a.C = C; a.P = P;
    set_layout(a, layout);
    const bool tok = layout == JIRF_LAYOUT_TOKENS;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Scope sc("train_residual_norm", 10.0 * B * C * (double)P, (dtype == JIRF_F32 ? 4.0 : 2.0) * B * C * (double)P * (pre_kind ? 4 : 3), s);
    RN_DISPATCH(dtype, tok, rn_fwd_sweep, dim3(sweep_grid(tok, B, P)), dim3(256), s, a);
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

long jirf_train_residual_norm_bwd_work_floats(int dtype, int layout, int post_kind, int gate_kind, int pre_kind, int B, int C, int P) {
  if (!dtype_ok(dtype) || (layout != JIRF_LAYOUT_PLANAR && layout != JIRF_LAYOUT_TOKENS) || !kind_ok(post_kind) ||
      !kind_ok(pre_kind) || gate_kind < 0 || gate_kind > 2 || B <= 0 || C <= 0 || P <= 0)
    return -1;
  RnArgs a{};
  a.post = post_kind; a.pre = pre_kind; a.gate_kind = gate_kind; a.B = B; a.C = C; a.P = P;
  bwd_workers(a);
  return bwd_work(a).total;
}

int jirf_train_residual_norm_bwd(const void* dy, long dy_bs, const void* dn, long dn_bs, const void* y, long y_bs, const void* f,
                                 long f_bs, const float* stats, int dtype, int layout, int post_kind, const float* post_w,
                                 const float* post_b, int gate_kind, const float* gate, const float* scale, int pre_kind,
                                 const float* pre_w, void* dx, long dx_bs, void* df, long df_bs, float* dpost_w, float* dpost_b,
                                 float* dgate, float* dpre_w, float* dpre_b, int accumulate, float* work, int B, int C, int P,
                                 void* stream) {
  return guarded_r([&] {
    const char* who = "residual_norm_bwd";
    check_common(who, dtype, layout, post_kind, post_w, gate_kind, gate, pre_kind, pre_w, B, C, P);
    JIRF_REQUIRE(dx && df && (dy || pre_kind), JIRF_EINVAL, "%s: null activation gradient", who);
    JIRF_REQUIRE(!pre_kind || (dn && y), JIRF_EINVAL, "%s: the norm before the next block needs dn and y", who);
    JIRF_REQUIRE(!(post_kind || gate_kind) || f, JIRF_EINVAL, "%s: a norm or gate on the branch needs f", who);
    JIRF_REQUIRE(!(post_kind || pre_kind) || stats, JIRF_EINVAL, "%s: a norm needs the forward's statistics", who);
    JIRF_REQUIRE((!dpost_w || post_kind) && (!dpost_b || post_kind == 1) && (!dgate || gate_kind) && (!dpre_w || pre_kind) &&
                     (!dpre_b || pre_kind == 1),
                 JIRF_EINVAL, "%s: a parameter gradient without its norm or gate", who);
    JIRF_REQUIRE(!(dpost_w || dpost_b || dgate || dpre_w || dpre_b || pre_kind) || work, JIRF_EINVAL, "%s: null work", who);
    RnArgs a{};
    a.dy = dy; a.dn = dn; a.y_in = y; a.f = f; a.dx = dx; a.df = df;
    a.dy_bs = batch_stride(who, "dy", dy, dy_bs, dtype, B, C, P);
    a.dn_bs = batch_stride(who, "dn", dn, dn_bs, dtype, B, C, P);
    a.yi_bs = batch_stride(who, "y", y, y_bs, dtype, B, C, P);
    a.f_bs = batch_stride(who, "f", f, f_bs, dtype, B, C, P);
    a.dx_bs = batch_stride(who, "dx", dx, dx_bs, dtype, B, C, P);
    a.df_bs = batch_stride(who, "df", df, df_bs, dtype, B, C, P);
    const Span ins[] = {{"dy", dy, a.dy_bs}, {"dn", pre_kind ? dn : nullptr, a.dn_bs}, {"y", pre_kind ? y : nullptr, a.yi_bs},
                        {"f", post_kind || gate_kind ? f : nullptr, a.f_bs}};
    const Span sdx{"dx", dx, a.dx_bs}, sdf{"df", df, a.df_bs};
    for (const Span& in : ins) {
      check_apart(who, sdx, in, dtype, B, C, P, false);
      check_apart(who, sdf, in, dtype, B, C, P, false);
    }
    check_apart(who, sdx, sdf, dtype, B, C, P, false);
    a.post = post_kind; a.pre = pre_kind; a.gate_kind = gate_kind;
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.gate = gate; a.scale = scale;
    a.stats_in = stats; a.accumulate = accumulate; a.B = B; a.C = C; a.P = P;
    set_layout(a, layout);
    bwd_workers(a);
    const BwdWork wk = bwd_work(a);
    a.rowsum = work;
    a.part = work + wk.rowsum;
    a.part_gate = a.part + wk.part;
    a.dgate = dgate;
    const bool tok = layout == JIRF_LAYOUT_TOKENS;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int reads = 1 + (pre_kind ? 2 : 0) + (post_kind || gate_kind ? 1 : 0);
    Scope sc("train_residual_norm_bwd", 25.0 * B * C * (double)P, (dtype == JIRF_F32 ? 4.0 : 2.0) * B * C * (double)P * (reads + 2), s);
    RN_DISPATCH(dtype, tok, rn_bwd_sweep, dim3(sweep_grid(tok, B, P)), dim3(256), s, a);
    if (dpost_w || dpost_b || dgate || dpre_w || dpre_b) {
      const long workers = n_workers(a);
      RN_DISPATCH(dtype, tok, rn_bwd_params_sweep, dim3((unsigned)((C + (tok ? 63 : 3)) / (tok ? 64 : 4)), (unsigned)workers), dim3(256), s, a);
      ReduceArgs r{};
      float* outs[Q_N] = {dpost_w, dpost_b, gate_kind == 1 ? dgate : nullptr, dpre_w, dpre_b};
      int nq = 0;
      for (int q = 0; q < Q_N; ++q)
        if (outs[q]) {
          r.part[nq] = a.part + (long)q * workers * C;
          r.out[nq++] = outs[q];
        }
      r.rows = workers; r.C = C; r.accumulate = accumulate;
      if (nq) hipLaunchKernelGGL(rn_reduce, dim3((unsigned)((C + 31) / 32), nq, 1), dim3(1024), 0, s, r);
      if (gate_kind == 2 && dgate && a.S > 1) {
        ReduceArgs g{};
        g.part[0] = a.part_gate;
        g.out[0] = dgate;
        g.rows = a.S; g.C = C; g.accumulate = accumulate;
        hipLaunchKernelGGL(rn_reduce, dim3((unsigned)((C + 31) / 32), 1, (unsigned)B), dim3(1024), 0, s, g);
      }
    }
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

}  // extern "C"
