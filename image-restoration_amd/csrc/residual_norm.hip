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
#include <climits>
#include <cmath>

#include "residual_norm.h"

namespace jirf {
namespace {

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
// Channel indices are 32 bits and step up to 256 past the last channel.
constexpr int RN_MOST_C = INT_MAX - 511;
// The launches that sum the parameter gradients have up to 64 threads per channel (RED_C columns of RED_R rows; planar, four
// channels of 256 threads), and a grid holds fewer than 2^32 threads.
constexpr int RN_MOST_C_PARAMS = (1 << 26) - 16;

void check_common(const char* who, int dtype, int layout, int post, const float* post_w, int gate_kind, const float* gate, int pre,
                  const float* pre_w, int B, int C, int P) {
  JIRF_REQUIRE(dtype_ok(dtype), JIRF_EINVAL, "%s: dtype %d (only fp32, bf16 and fp16)", who, dtype);
  JIRF_REQUIRE(layout == JIRF_LAYOUT_PLANAR || layout == JIRF_LAYOUT_TOKENS, JIRF_EINVAL, "%s: layout %d", who, layout);
  JIRF_REQUIRE(kind_ok(post) && kind_ok(pre) && gate_kind >= 0 && gate_kind <= 2, JIRF_EINVAL,
               "%s: norm kinds are 0..3 and gate kinds 0..2, got post %d, pre %d, gate %d", who, post, pre, gate_kind);
  JIRF_REQUIRE((!post || post_w) && (!pre || pre_w) && (!gate_kind || gate), JIRF_EINVAL,
               "%s: a norm without its weight or a gate without its factors", who);
  JIRF_REQUIRE(B > 0 && C > 0 && P > 0, JIRF_EINVAL, "%s: sizes B %d C %d P %d", who, B, C, P);
  JIRF_REQUIRE(C <= RN_MOST_C, JIRF_EINVAL, "%s: %d channels, at most %d", who, C, RN_MOST_C);
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

#define RN_TYPE(dtype, CALL)                          \
  do {                                                \
    if (dtype == JIRF_F32) CALL<float> RN_ARGS;       \
    else if (dtype == JIRF_BF16) CALL<__bf16> RN_ARGS; \
    else CALL<_Float16> RN_ARGS;                      \
  } while (0)

// Which kernel serves (layout, type, B, C, P): the register form wherever a workgroup of 512 threads can hold a token (or a
// few pixels) of all channels, the sweep form beyond.
RnForm choose_form(RnArgs& a, int dtype, int layout, bool backward) {
  RnForm f{};
  f.tok = layout == JIRF_LAYOUT_TOKENS;
  const int vec = f.tok ? (dtype == JIRF_F32 ? 4 : 8) : 4;
  a.tiles = a.P;
  a.S = a.ipw = 1;
  f.threads = 256;
  long per_block = 1;                  // workers of a workgroup
  const long image_bytes = (long)a.C * a.P * (dtype == JIRF_F32 ? 4 : 2);
  if ((f.tok ? a.C : a.P) < vec || image_bytes >= 1l << 32) {
    f.lanes = -1;
  } else if (f.tok) {
    // Eight channels per thread, in groups of lanes that share a wave up to 512 channels (22 channels: groups of four lanes
    // against eight, backward of 524288 tokens fp32 67 / 73 us, bf16 52 / 71 us).  Sixteen where eight would need more than
    // 512 threads; in the backward of 16-bit types from 2049 channels on, half as many waves (2x6464x2163 fp16 113 us
    // against 126 with eight, 4x1066x3344 29 / 32).  Not where that loses: fp32 (2x3464x2600 88 / 84 us), no norm and no gate
    // on the branch (8x1066x4096 bf16 73 / 65), a gate per image, whose sums close with every image: short images lose more
    // (16x300x4096 bf16 82 / 70, 64x37x2300 71 / 67) than long ones gain (2x6464x2600 fp16 125 / 129).
    const int threads8 = (a.C + 7) / 8;
    const bool wide16 = backward && dtype != JIRF_F32 && a.gate_kind != 2 && (a.post || a.gate_kind);
    f.nv = 8 / vec;
    if (threads8 <= 64) {
      f.lanes = threads8 <= 4 ? 4 : threads8 <= 8 ? 8 : threads8 <= 16 ? 16 : threads8 <= 32 ? 32 : 64;
      f.threads = 256;
      per_block = f.threads / f.lanes;
    } else if (threads8 <= (wide16 ? 256 : 512)) {
      f.threads = (threads8 + 63) / 64 * 64;
    } else if (a.C <= 8192) {
      f.nv *= 2;
      f.threads = ((a.C + 15) / 16 + 63) / 64 * 64;
    } else {
      f.lanes = -1;
    }
  } else {
    // four channels of four pixels per thread: as many pixel lanes (of 32) as the channels leave room for in 256 threads,
    // more threads only to keep eight lanes (a 128-byte line of fp32: backward of 4x256x16384 with 512 threads 109 us, with
    // four lanes in 256 threads 131 us), or fewer lanes than that to fit at all.  The 16-bit forward has registers for 1024
    // threads (3x567x49959 bf16 272 us; with 512 at most 382 us).
    // Eight channels of four pixels in the fp32 forward where eight lanes of four would need more than 256 threads, which keeps
    // eight lanes up to 512 channels and four up to 1024: 4x512x16384 182 -> 133 us, 4x300x16384 91 -> 68, 4x256x16384
    // 57 -> 50, 4x700x16384 251 -> 232; 4x128x16384 would lose (25.7 -> 26.2).  Not below 256 tiles while four channels keep
    // four lanes (8x140x300 5.1 -> 6.7).  The backward and the 16-bit forward gain at some sizes and lose at others
    // (backward without a branch norm 4x300x16384 104 -> 100, 12x256x4096 50 -> 61; with one it spills some 190 registers;
    // bf16 4x256x16384 39 -> 35, 4x200x16384 27 -> 29).
    const int most = !backward && dtype != JIRF_F32 ? 1024 : 512;
    const bool eight = !backward && dtype == JIRF_F32 && a.C > 128 && (a.C > 512 || ((long)a.P + 31) / 32 * a.B >= 256);
    f.nv = eight ? 8 : 4;
    const int rows = (a.C + f.nv - 1) / f.nv;
    f.lanes = 32;
    while (f.lanes > 8 && f.lanes * rows > 256) f.lanes >>= 1;
    while (f.lanes > 2 && f.lanes * rows > most) f.lanes >>= 1;
    // no wider than the plane, and narrower while the tiles leave CUs idle
    while (f.lanes > 4 && (f.lanes * 2 >= a.P || ((long)a.P + f.lanes * 4 - 1) / (f.lanes * 4) * a.B < 256)) f.lanes >>= 1;
    f.threads = std::max(64, (f.lanes * rows + 63) / 64 * 64);
    if (f.threads > most) f.lanes = -1;
    else a.tiles = (int)(((long)a.P + f.lanes * 4 - 1) / (f.lanes * 4));
  }
  // Operands that the 256 MB cache cannot hold between their producer and this call are read past it, where a row is some
  // kilobytes: tokens 2x8192x2048 fp32 forward 4.99 -> 6.24 TB/s, 4x4096x2048 bf16 backward 4.4 -> 4.9; smaller ones
  // lose (8000x1000 fp32 6.0 -> 5.9, 2x4096x1024 bf16 5.0 -> 4.3), and so do narrow pieces of planar rows.
  // Outputs beyond it go past it too in the forward (8x4096x4096 bf16 5.0 -> 5.5 TB/s; below that 5.9 -> 5.3).
  const int tensors = backward ? (a.pre ? 4 : 2) + (a.post || a.gate_kind ? 2 : 1) : a.pre ? 4 : 3;
  const long bytes = image_bytes * a.B, cache = 256l << 20;
  f.stream = !f.tok || f.lanes != 0 || bytes * tensors <= cache ? 0 : !backward && bytes * (a.pre ? 2 : 1) > cache ? 2 : 1;
  // Workers.  Workgroups of a kernel that loops over its tiles are best all resident at once (256 CUs, and a CU holds 8 waves
  // of the backward's 256 registers, 16 and more of the forward's); more and smaller ones only while they are small.  Tokens
  // 4x4096x2048 bf16 backward (256 threads): 256 / 512 / 1024 workgroups 143 / 94 / 108 us; 4x1066x3344 fp16: 512 threads
  // 37 / 41 / 51 us; tokens 19061x2905 fp16 forward (384 threads): 512 / 768 / 1024 90 / 73 / 95 us; planar 13x153x21471
  // fp16 forward (320 threads): 512 / 1024 / 2048 114 / 141 / 132 us.  In the backward each also leaves a row of partial
  // sums.
  if (f.lanes < 0) a.tiles = (int)(((long)a.P + 63) / 64);
  long want = 256;
  if (f.lanes >= 0) {
    if (backward) want = 256 * std::max(1, 512 / f.threads);
    else if (f.tok && f.lanes == 0 && f.threads >= 256) want = 256 * (1152 / f.threads);
    else want = f.threads <= 256 ? 2048 : f.threads <= 512 ? 512 : 256;
  }
  want *= per_block;
  if (a.B >= want) {
    a.ipw = (int)((a.B + want - 1) / want);
  } else {
    // the same number of tiles for every worker, but the last few
    const long S = std::max<long>(1, std::min<long>(a.tiles, want / a.B)), rounds = (a.tiles + S - 1) / S;
    a.S = (int)((a.tiles + rounds - 1) / rounds);
  }
  const long workers = a.S > 1 ? (long)a.B * a.S : ((long)a.B + a.ipw - 1) / a.ipw;
  f.blocks = (unsigned)((workers + per_block - 1) / per_block);
  a.part_rows = f.blocks;
  return f;
}

struct BwdWork {
  long rowsum, part, part_gate, total;   // floats
};
BwdWork bwd_work(const RnArgs& a, const RnForm& f) {
  BwdWork w{};
  w.rowsum = f.lanes < 0 && a.pre ? 2l * a.B * a.P : 0;
  w.part = (long)RN_Q_N * a.part_rows * a.C;
  w.part_gate = a.gate_kind == 2 && a.S > 1 ? (long)a.B * a.S * a.C : 0;
  w.total = w.rowsum + w.part + w.part_gate;
  return w;
}

// Adds the partial sums up, rows in order per thread and the row lanes in order, in 64 bits.  blockIdx.y 0: the branch (G1,
// G0 -> dpost_w, dpost_b, dgate), 1: the norm before the next block, 2 + b: image b's gate from its S workers.
struct ReduceArgs {
  const float* part;
  long rows, C;
  float *dpost_w, *dpost_b, *dgate, *dpre_w, *dpre_b;
  const float *gate, *post_w, *post_b;   // gate: null with a gate per image (its factors are in the sums already)
  int has_post, accumulate;
  const float* part_gate;                // [B][S][C], for dgate_image [B][C]
  float* dgate_image;
  long S;
};
// Sums of column c of two planes (r null: none) over the rows: 64 row lanes of 16 columns, eight loads of each in flight.
constexpr int RED_C = 16, RED_R = 64;
template <bool TWO>
__device__ __forceinline__ void reduce_columns(const float* q, const float* r, long rows, long C, long c, double (*red)[RED_C + 1],
                                               double& vq, double& vr) {
  const int cl = threadIdx.x % RED_C, rl = threadIdx.x / RED_C;
  double t[2] = {0.0, 0.0};
  if (c < C) {
    constexpr int U = 8;
    for (long i = rl; i < rows; i += U * RED_R) {
      float x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long k = min(i + u * RED_R, rows - 1) * C + c;
        x[u] = q[k];
        y[u] = TWO ? r[k] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = i + u * RED_R < rows;
        t[0] += on ? (double)x[u] : 0.0;
        if (TWO) t[1] += on ? (double)y[u] : 0.0;
      }
    }
  }
  double v[2] = {0.0, 0.0};
#pragma unroll
  for (int k = 0; k < (TWO ? 2 : 1); ++k) {
    __syncthreads();
    red[rl][cl] = t[k];
    __syncthreads();
    if (rl == 0)
#pragma unroll 16
      for (int i = 0; i < RED_R; ++i) v[k] += red[i][cl];
  }
  vq = v[0];
  vr = v[1];
}
__device__ __forceinline__ void reduce_out(float* out, long c, double v, int accumulate) {
  if (out) out[c] = accumulate ? (float)((double)out[c] + v) : (float)v;
}
__global__ __launch_bounds__(RED_C * RED_R) void rn_reduce(const ReduceArgs a) {
  __shared__ double red[RED_R][RED_C + 1];
  const long c = (long)blockIdx.x * RED_C + threadIdx.x % RED_C;
  const bool writer = threadIdx.x < RED_C && c < a.C;
  const long plane = a.rows * a.C;
  double v0, v1;
  if (blockIdx.y == 0) {
    if (!a.dpost_w && !a.dpost_b && !a.dgate) return;
    const float *g1 = a.part + RN_Q_G1 * plane, *g0 = a.part + RN_Q_G0 * plane;
    const bool g1_used = a.dpost_w || a.dgate, g0_used = a.dpost_b || (a.dgate && a.post_b);
    if (g1_used && g0_used) {
      reduce_columns<true>(g1, g0, a.rows, a.C, c, red, v0, v1);
    } else {
      reduce_columns<false>(g1_used ? g1 : g0, nullptr, a.rows, a.C, c, red, v0, v1);
      if (!g1_used) v1 = v0;
    }
    if (!writer) return;
    const double g = a.gate ? (double)a.gate[c] : 1.0;
    reduce_out(a.dpost_w, c, g * v0, a.accumulate);
    reduce_out(a.dpost_b, c, g * v1, a.accumulate);
    reduce_out(a.dgate, c, a.has_post ? a.post_w[c] * v0 + (a.post_b ? a.post_b[c] * v1 : 0.0) : v0, a.accumulate);
  } else if (blockIdx.y == 1) {
    if (!a.dpre_w && !a.dpre_b) return;
    const float *w = a.part + RN_Q_PRE_W * plane, *b = a.part + RN_Q_PRE_B * plane;
    if (a.dpre_w && a.dpre_b) {
      reduce_columns<true>(w, b, a.rows, a.C, c, red, v0, v1);
    } else {
      reduce_columns<false>(a.dpre_w ? w : b, nullptr, a.rows, a.C, c, red, v0, v1);
      v1 = v0;
    }
    if (!writer) return;
    reduce_out(a.dpre_w, c, v0, a.accumulate);
    reduce_out(a.dpre_b, c, v1, a.accumulate);
  } else {
    const long b = blockIdx.y - 2;
    reduce_columns<false>(a.part_gate + b * a.S * a.C, nullptr, a.S, a.C, c, red, v0, v1);
    if (writer) reduce_out(a.dgate_image + b * a.C, c, v0, a.accumulate);
  }
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    Scope sc("train_residual_norm", 10.0 * B * C * (double)P, (dtype == JIRF_F32 ? 4.0 : 2.0) * B * C * (double)P * (pre_kind ? 4 : 3), s);
    const RnForm f_ = choose_form(a, dtype, layout, false);
#define RN_ARGS (a, f_, s)
    RN_TYPE(dtype, rn_launch_fwd);
#undef RN_ARGS
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

long jirf_train_residual_norm_bwd_work_floats(int dtype, int layout, int post_kind, int gate_kind, int pre_kind, int B, int C, int P) {
  if (!dtype_ok(dtype) || (layout != JIRF_LAYOUT_PLANAR && layout != JIRF_LAYOUT_TOKENS) || !kind_ok(post_kind) ||
      !kind_ok(pre_kind) || gate_kind < 0 || gate_kind > 2 || B <= 0 || C <= 0 || C > RN_MOST_C || P <= 0)
    return -1;
  RnArgs a{};
  a.post = post_kind; a.pre = pre_kind; a.gate_kind = gate_kind; a.B = B; a.C = C; a.P = P;
  const RnForm form = choose_form(a, dtype, layout, true);
  return bwd_work(a, form).total;
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
    JIRF_REQUIRE((dx || !pre_kind) && df && (dy || pre_kind), JIRF_EINVAL, "%s: null activation gradient", who);
    JIRF_REQUIRE(!pre_kind || (dn && y), JIRF_EINVAL, "%s: the norm before the next block needs dn and y", who);
    JIRF_REQUIRE(!(post_kind || gate_kind) || f, JIRF_EINVAL, "%s: a norm or gate on the branch needs f", who);
    JIRF_REQUIRE(!(post_kind || pre_kind) || stats, JIRF_EINVAL, "%s: a norm needs the forward's statistics", who);
    JIRF_REQUIRE((!dpost_w || post_kind) && (!dpost_b || post_kind == 1) && (!dgate || gate_kind) && (!dpre_w || pre_kind) &&
                     (!dpre_b || pre_kind == 1),
                 JIRF_EINVAL, "%s: a parameter gradient without its norm or gate", who);
    const bool params = dpost_w || dpost_b || dgate || dpre_w || dpre_b;
    JIRF_REQUIRE(!(params || pre_kind) || work, JIRF_EINVAL, "%s: null work", who);
    JIRF_REQUIRE(!params || C <= RN_MOST_C_PARAMS, JIRF_EINVAL, "%s: parameter gradients of %d channels, at most %d", who, C, RN_MOST_C_PARAMS);
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
    const RnForm form = choose_form(a, dtype, layout, true);
    const BwdWork wk = bwd_work(a, form);
    const bool branch = post_kind || gate_kind;
    if (work) {
      a.rowsum = work;
      a.part = params ? work + wk.rowsum : nullptr;
      a.part_gate = dgate ? work + wk.rowsum + wk.part : nullptr;
    }
    a.dgate = gate_kind == 2 ? dgate : nullptr;
    const bool gate1 = gate_kind == 1 && dgate;
    a.wanted = (dpost_w || gate1 ? 1 << RN_Q_G1 : 0) | (dpost_b || (gate1 && post_kind == 1 && post_b) ? 1 << RN_Q_G0 : 0) |
               (dpre_w ? 1 << RN_Q_PRE_W : 0) | (dpre_b ? 1 << RN_Q_PRE_B : 0);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int reads = 1 + (pre_kind ? 2 : 0) + (branch ? 1 : 0);
    const int mode = !branch ? RN_BWD_STREAM : gate_kind == 2 ? RN_BWD_IMAGE_GATE : RN_BWD_BRANCH;
    Scope sc("train_residual_norm_bwd", 25.0 * B * C * (double)P, (dtype == JIRF_F32 ? 4.0 : 2.0) * B * C * (double)P * (reads + 2), s);
#define RN_ARGS (a, form, mode, params, s)
    RN_TYPE(dtype, rn_launch_bwd);
#undef RN_ARGS
    if (params) {
      const bool images = gate_kind == 2 && dgate && a.S > 1;
      const ReduceArgs r{a.part, a.part_rows, C, dpost_w, dpost_b, gate_kind == 1 ? dgate : nullptr, dpre_w, dpre_b,
                         gate_kind == 1 ? gate : nullptr, post_w, post_kind == 1 ? post_b : nullptr, post_kind, accumulate,
                         images ? a.part_gate : nullptr, images ? dgate : nullptr, a.S};
      // (S > 1 only below a few thousand images)
      hipLaunchKernelGGL(rn_reduce, dim3((unsigned)((C + RED_C - 1) / RED_C), images ? 2u + B : 2u), dim3(RED_C * RED_R), 0, s, r);
    }
    JIRF_HIP_CHECK(hipGetLastError());
    return JIRF_OK;
  });
}

}  // extern "C"
