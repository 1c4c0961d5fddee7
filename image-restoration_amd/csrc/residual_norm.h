// Kernels of the residual join with its norms (formulas in residual_norm.hip), as templates over the activation type:
// residual_norm_{f32,bf16,f16}.hip instantiate them, residual_norm.hip chooses among them.
#pragma once

#include "runtime.h"

namespace jirf {

struct RnArgs {
  // activations, element (b, c, p) at ptr + b * bs + c * cs + p * ps
  const void *x, *f, *dy, *dn, *y_in;
  void *y, *n, *dx, *df;
  long x_bs, f_bs, dy_bs, dn_bs, yi_bs, y_bs, n_bs, dx_bs, df_bs;
  long cs, ps;
  const float *post_w, *post_b, *gate, *scale, *pre_w, *pre_b;
  const float* stats_in;   // [4][B][P]
  float* stats;            // [4][B][P] or null
  float* rowsum;           // backward of the sweep form: [2][B][P], the two row means of the pre norm's gradient
  float* part;             // backward: [4][part_rows][C] partial sums, RN_Q_*
  float* part_gate;        // backward, gate kind 2 and S > 1: [B][S][C]
  float* dgate;            // backward, gate kind 2 and S == 1: written directly
  long part_rows;
  int wanted;              // bit q: the sums RN_Q_* q are needed
  int post, pre, gate_kind, accumulate;
  float eps;
  int B, C, P;
  // Workers: S per image, each with every S-th tile (ipw == 1), or one per ipw images (S == 1).
  int S, ipw, tiles;
};
// The branch's parameter gradients come from two sums per channel, G1 = sum s dyt vh and G0 = sum s dyt (vh = the
// normalised f, or f): dpost_w = gate G1, dpost_b = gate G0, dgate = post_w G1 + post_b G0 (or G1 without a norm).
// With a gate per image the factors belong inside the sum over the images: then the sums are dpost_w and dpost_b.
enum { RN_Q_G1 = 0, RN_Q_G0 = 1, RN_Q_PRE_W = 2, RN_Q_PRE_B = 3, RN_Q_N = 4 };

// Which kernel serves a call.  lanes: tokens - threads per token (4..64, several tokens per wave) or 0 (the whole
// workgroup); planar - pixel lanes; -1: the sweep form.
struct RnForm {
  bool tok;
  int stream;              // 1: operands larger than the caches are read past them, 2: outputs written past them too
  int lanes, nv, threads;
  unsigned blocks;
};
enum { RN_BWD_STREAM = 0, RN_BWD_BRANCH = 1, RN_BWD_IMAGE_GATE = 2 };

template <typename T> void rn_launch_fwd(const RnArgs& a, const RnForm& f, hipStream_t s);
template <typename T> void rn_launch_bwd(const RnArgs& a, const RnForm& f, int mode, bool params, hipStream_t s);

}  // namespace jirf

#ifdef JIRF_RN_KERNELS
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

// VEC consecutive elements, read and written at the alignment of one element (rows of odd length, channel slices: the
// memory instructions take any 2- or 4-byte address), `off` bytes into an image.
// NT: not kept in the caches.
template <typename T, int VEC, bool NT> struct Pack {
  typedef T V __attribute__((ext_vector_type(VEC)));
  typedef T VU __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  V v;
  __device__ __forceinline__ void load(const char* image, unsigned off) {
    const VU* p = reinterpret_cast<const VU*>(image + off);
    v = NT ? __builtin_nontemporal_load(p) : *p;
  }
  __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
};
template <typename T, int VEC, bool NT = false>
__device__ __forceinline__ void store_vec(char* image, unsigned off, const float* f) {
  typedef T V __attribute__((ext_vector_type(VEC)));
  typedef T VU __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = (T)f[i];
  if (NT) __builtin_nontemporal_store(v, reinterpret_cast<VU*>(image + off));
  else *reinterpret_cast<VU*>(image + off) = v;
}
// the last `own` of VEC values
template <typename T, int VEC>
__device__ __forceinline__ void store_some(char* image, unsigned off, int own, const float* f) {
  if (own == VEC) {
    store_vec<T, VEC>(image, off, f);
  } else {
    T* p = reinterpret_cast<T*>(image + off);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= VEC - own) p[i] = (T)f[i];
  }
}

constexpr int RN_T = 512;         // most threads of a workgroup in the register form (256 registers each)
constexpr int RN_T16 = 1024;      // the same for the planar forward of 16-bit types (128 registers each)
constexpr int RN_LANE_T = 256;    // threads of a workgroup whose waves hold several tokens each

// x + the value of another lane, by one data-parallel instruction (no LDS access, as a shuffle makes).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_row16(float x) {       // rows of 16 lanes, in pairs
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_half32(float x) {      // the two halves of the wave
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The sum over the lanes i, i + STRIDE, i + 2 STRIDE, ... of a group of SIZE lanes, in every one of them.
template <int STRIDE, int SIZE>
__device__ __forceinline__ float lane_sum(float x) {
  if constexpr (SIZE == 4 || SIZE == 8) {
    static_assert(STRIDE == 1, "");
    x = add_dpp<0xB1>(x);                                   // lane ^ 1
    x = add_dpp<0x4E>(x);                                   // lane ^ 2
    if constexpr (SIZE == 8) x = add_dpp<0x141>(x);         // lane 7 - i of the eight: the other four's sum
  } else {
    if constexpr (STRIDE <= 8) x = add_dpp<0x128>(x);       // rotations inside the row of 16
    if constexpr (STRIDE <= 4) x = add_dpp<0x124>(x);
    if constexpr (STRIDE <= 2) x = add_dpp<0x122>(x);
    if constexpr (STRIDE <= 1) x = add_dpp<0x121>(x);
    if constexpr (SIZE >= 32 && STRIDE <= 16) x = add_row16(x);
    if constexpr (SIZE >= 64) x = add_half32(x);
  }
  return x;
}
// 1 / sqrt(x) within half a unit in the last place and 2^-21 of one: the hardware's estimate and one Newton step whose residual
// 1 - x y^2 keeps the product's remainder.  Nearly always the nearest value: of the 2^24 in [1, 4), 1 to 7 get the other
// neighbour, depending on which value within one unit the estimate is (2.1552868 from the nearest estimate, for one).  Small x are
// scaled into the estimate's range, 0 and infinity are as they are.
__device__ __forceinline__ float recip_sqrt(float x) {
  const bool tiny = x < 0x1p-96f;
  x *= tiny ? 0x1p64f : 1.0f;
  const float y = __builtin_amdgcn_rsqf(x), p = x * y, lo = fmaf(x, y, -p);
  const float e = fmaf(-lo, y, fmaf(-p, y, 1.0f)), r = fmaf(0.5f * y, e, y);
  return (y > 0.f && y < __builtin_inff() ? r : y) * (tiny ? 0x1p32f : 1.0f);
}

// ---- a tile in registers ------------------------------------------------------------------------------------------------
// A worker owns a set of tiles; every thread holds NV vectors of VEC elements of each operand of a tile, so an operand is
// read once.  tokens: a tile is one token, a vector VEC consecutive channels, and the token's threads are L lanes of a
// wave (a worker per lane group) or the workgroup (L == 0).  planar: a tile is L * VEC pixels of all channels, a vector VEC
// consecutive pixels of one channel; L lanes run along the pixels, the other threads along the channels.
// A vector that would reach past the channels (the pixels) is moved back to end at the last one, so every load is whole and
// none branches; the elements it then shares with its neighbour belong to the neighbour: they are left out of sums and
// stores.  A thread without a channel repeats the last one and owns nothing.  Needs C >= VEC (tokens) or P >= VEC (planar),
// and less than 2^32 bytes in an image.
template <typename T, bool TOK, int L, int NV, int VEC, int NT>
struct Tile {
  static constexpr int NS = TOK ? 1 : VEC;       // statistics per thread: its token's, or one per pixel of its vector
  static constexpr int NP = TOK ? VEC : 1;       // parameters per vector
  typedef Pack<T, VEC, (NT > 0)> Vec;
  const RnArgs& a;
  float* red;                                    // LDS of two reductions
  int buf;
  int ch, nch, pl;                               // position among the token's threads, their number, pixel lane
  int own[NV];                                   // tokens: elements of each vector that are its own; planar: 1 or 0
  unsigned off[NV];                              // bytes from the token's first channel / from the image's first pixel 0

  // two buffers of [waves][token lanes][two sums per statistic]
  static constexpr int RED = TOK ? (L ? 1 : 2 * (RN_T / 64) * 2) : 2 * (RN_T16 / 64) * L * 2 * VEC;

  __device__ __forceinline__ Tile(const RnArgs& args, float* lds) : a(args), red(lds), buf(0) {
    const int tid = threadIdx.x;
    if (TOK) {
      ch = L ? tid & (L - 1) : tid;
      nch = L ? L : (int)blockDim.x;
      pl = 0;
    } else {
      pl = tid & (L - 1);
      ch = tid / L;
      nch = blockDim.x / L;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (TOK) {
        const int c = (j * nch + ch) * VEC;
        own[j] = max(0, min(VEC, a.C - c));
        off[j] = (unsigned)channel(j) * sizeof(T);
      } else {
        own[j] = j * nch + ch < a.C;
        off[j] = (unsigned)channel(j) * (unsigned)a.P * (unsigned)sizeof(T);
      }
    }
  }
  // first channel of vector j as loaded
  __device__ __forceinline__ int channel(int j) const {
    return TOK ? min((j * nch + ch) * VEC, a.C - VEC) : min(j * nch + ch, a.C - 1);
  }
  __device__ __forceinline__ bool exists(int j, int v) const { return TOK ? v >= VEC - own[j] : own[j] != 0; }
  // whether an element of a tile with px own pixels is the thread's own
  __device__ __forceinline__ bool mine(int j, int v, int px) const { return exists(j, v) && (TOK || v >= VEC - px); }
  // first pixel of this lane's vector in tile t as loaded, and how many (the last ones) are its own
  __device__ __forceinline__ int pixel(int t) const { return TOK ? t : (int)min(((long)t * L + pl) * VEC, (long)a.P - VEC); }
  __device__ __forceinline__ int own_pixels(int t) const {
    return TOK ? 1 : (int)max(0l, min((long)VEC, (long)a.P - ((long)t * L + pl) * VEC));
  }
  __device__ __forceinline__ unsigned start(int t) const {
    return (TOK ? (unsigned)t * (unsigned)a.C : (unsigned)pixel(t)) * (unsigned)sizeof(T);
  }
  static __device__ __forceinline__ const char* image(const void* p, long bs, int b) {
    return reinterpret_cast<const char*>(static_cast<const T*>(p) + b * bs);
  }
  __device__ __forceinline__ void load(const char* img, unsigned st, Vec (&r)[NV]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j].load(img, st + off[j]);
  }
  // whether some vector of tile t is shared (the same answer for the whole workgroup)
  __device__ __forceinline__ bool edge(int t) const { return TOK ? a.C % VEC != 0 : (long)(t + 1) * (L * VEC) > a.P; }
  __device__ __forceinline__ void store(void* p, long bs, int b, int t, const float (&f)[NV][VEC]) const {
    char* img = const_cast<char*>(image(p, bs, b));
    const unsigned st = start(t);
    if (!edge(t)) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (own[j]) store_vec<T, VEC, NT == 2>(img, st + off[j], f[j]);
    } else {
      const int px = own_pixels(t);
#pragma unroll
      for (int j = 0; j < NV; ++j) store_some<T, VEC>(img, st + off[j], TOK ? own[j] : own[j] ? px : 0, f[j]);
    }
  }
  // a [C] array in the thread's channels; `none` for a channel that is not its own, or without an array
  __device__ __forceinline__ void params(const float* p, float none, float (&r)[NV][NP]) const {
    typedef float F __attribute__((ext_vector_type(NP), aligned(4)));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int v = 0; v < NP; ++v) r[j][v] = none;
      if (!p) continue;
      if constexpr (NP == 1) {
        r[j][0] = own[j] ? p[channel(j)] : none;
      } else {
        const F q = *reinterpret_cast<const F*>(p + channel(j));
#pragma unroll
        for (int v = 0; v < NP; ++v) r[j][v] = exists(j, v) ? q[v] : none;
      }
    }
  }
  // Sums v[0..N) over the threads of the token.  Lanes first, then the waves in order through LDS; two buffers in turn, so
  // one barrier per reduction is enough.
  template <int N>
  __device__ __forceinline__ void reduce(float (&v)[N]) {
    constexpr int W = TOK ? 1 : L;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane_sum<W, TOK && L ? L : 64>(v[i]);
    if (TOK && L) return;
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (waves == 1) return;
    typedef float F __attribute__((ext_vector_type(N)));
    F* r = reinterpret_cast<F*>(red + buf * (RED / 2));
    buf ^= 1;
    F q;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = v[i];
    if (lane < W) r[wave * W + lane] = q;
    __syncthreads();
    const int at = TOK ? 0 : pl;
    q = r[at];
    for (int w = 1; w < waves; ++w) q += r[w * W + at];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = q[i];
  }
  // mean (0 for the root mean square) and reciprocal deviation, in two passes over the registers
  __device__ __forceinline__ void statistics(const float (&v)[NV][VEC], int kind, float (&mu)[NS], float (&rs)[NS]) {
    const float inv = 1.0f / (float)a.C;
#pragma unroll
    for (int s = 0; s < NS; ++s) mu[s] = 0.f;
    if (kind != 3) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (TOK || own[j])
#pragma unroll
          for (int i = 0; i < VEC; ++i) mu[TOK ? 0 : i] += !TOK || exists(j, i) ? v[j][i] : 0.f;
      reduce<NS>(mu);
#pragma unroll
      for (int s = 0; s < NS; ++s) mu[s] *= inv;
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) rs[s] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (TOK || own[j])
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = !TOK || exists(j, i) ? v[j][i] - mu[TOK ? 0 : i] : 0.f;
          rs[TOK ? 0 : i] = fmaf(d, d, rs[TOK ? 0 : i]);
        }
    reduce<NS>(rs);
#pragma unroll
    for (int s = 0; s < NS; ++s) rs[s] = recip_sqrt(fmaf(rs[s], inv, a.eps));
  }
  // Images [b0, b1) of worker w (none behind the last image), and its first tile in each: it takes every a.S-th from there.
  // There are at least a.S tiles, so every worker of an image has one.
  __device__ __forceinline__ void range(long w, int& b0, int& b1, int& t0) const {
    if (a.S > 1) {
      b0 = (int)min(w / a.S, (long)a.B);
      b1 = min(b0 + 1, a.B);
      t0 = (int)(w % a.S);
    } else {
      b0 = (int)min(w * a.ipw, (long)a.B);
      b1 = (int)min(w * a.ipw + a.ipw, (long)a.B);
      t0 = 0;
    }
  }
  // Workers are numbered along each XCD: neighbours, which share the cache lines at the tiles' edges (planar rows are rarely
  // whole lines, and a tile's piece of a row may be half of one), run at the same time on the same L2.
  __device__ __forceinline__ long worker() const {
    const long block = xcd_remap(blockIdx.x, gridDim.x);
    if (TOK && L) return block * (RN_LANE_T / (L ? L : 1)) + threadIdx.x / (L ? L : 1);
    return block;
  }
};

// Forward.  Reads x and f once and writes y and n once; the next tile's loads are issued before this tile's reductions.
// The branch's factors are folded: u = vh (gate w) + gate b.  Tokens 8x4096x4096 bf16 take 196 us
// (5.5 TB/s) and planar 2x32x65536 fp32 14.2 us (4.9 TB/s), the rate of a large copy; one token of 512 2.9 us, a launch.
// Furthest from the copy are planar 16-bit images of many channels (3x567x49959 bf16 272 us, 2.5 TB/s): there 32 bytes of a
// row fit beside the channels, and a barrier per reduction waits for up to 16 waves; which of the two costs more is not known.
template <typename T, bool TOK, int L, int NV, int VEC, int NT>
__global__ __launch_bounds__(TOK && L ? RN_LANE_T : !TOK && sizeof(T) == 2 ? RN_T16 : RN_T) void rn_fwd_tile(const RnArgs a) {
  typedef Tile<T, TOK, L, NV, VEC, NT> Ti;
  typedef typename Ti::Vec Vec;
  constexpr int NS = Ti::NS, NP = Ti::NP;
  // the next tile is fetched ahead where the registers (256 per thread) have room for two tiles
  constexpr bool PF = NV * VEC * sizeof(T) < 128;
  __shared__ __attribute__((aligned(32))) float lds[Ti::RED];
  Ti ti(a, lds);
  int b0, b1, t0;
  ti.range(ti.worker(), b0, b1, t0);
  const int t1 = a.tiles;
  if (b0 >= b1) return;                       // (uniform over the threads of a worker, and a worker's barriers are its own)
  float pw[NV][NP], pb[NV][NP], gw[NV][NP], gb[NV][NP];
  Vec xn[NV], fn[NV];
  if (PF) {
    ti.load(Ti::image(a.f, a.f_bs, b0), ti.start(t0), fn);
    ti.load(Ti::image(a.x, a.x_bs, b0), ti.start(t0), xn);
  }
  ti.params(a.pre ? a.pre_w : nullptr, 0.f, pw);
  ti.params(a.pre == 1 ? a.pre_b : nullptr, 0.f, pb);
  int gate_of = -1;
  for (int b = b0; b < b1; ++b) {
    if (gate_of < 0 || a.gate_kind == 2) {
      gate_of = b;
      ti.params(a.post ? a.post_w : nullptr, 1.f, gw);
      ti.params(a.post == 1 ? a.post_b : nullptr, 0.f, gb);
      if (a.gate_kind) {
        float g[NV][NP];
        ti.params(a.gate + (a.gate_kind == 2 ? (long)b * a.C : 0), 0.f, g);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            gw[j][i] *= g[j][i];
            gb[j][i] *= g[j][i];
          }
      }
    }
    const float s = a.scale ? a.scale[b] : 1.0f;
    for (int t = t0; t < t1; t += a.S) {
      if (!PF) {
        ti.load(Ti::image(a.f, a.f_bs, b), ti.start(t), fn);
        ti.load(Ti::image(a.x, a.x_bs, b), ti.start(t), xn);
      }
      Vec xv[NV], fv[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xv[j] = xn[j];
        fv[j] = fn[j];
      }
      const int bn = t + a.S < t1 ? b : b + 1, tn = t + a.S < t1 ? t + a.S : t0;
      if (PF && bn < b1) {
        ti.load(Ti::image(a.f, a.f_bs, bn), ti.start(tn), fn);
        ti.load(Ti::image(a.x, a.x_bs, bn), ti.start(tn), xn);
      }
      const int px = ti.own_pixels(t);
      float v[NV][VEC], mu0[NS], rs0[NS], mu1[NS], rs1[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) mu0[i] = rs0[i] = mu1[i] = rs1[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = fv[j].at(i);
      if (a.post) {
        ti.statistics(v, a.post, mu0, rs0);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[j][i] = (a.post == 1 ? v[j][i] - mu0[TOK ? 0 : i] : v[j][i]) * rs0[TOK ? 0 : i];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          v[j][i] = fmaf(s, fmaf(v[j][i], gw[j][TOK ? i : 0], gb[j][TOK ? i : 0]), xv[j].at(i));
      ti.store(a.y, a.y_bs, b, t, v);
      if (a.pre) {
        ti.statistics(v, a.pre, mu1, rs1);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            v[j][i] = fmaf((a.pre == 1 ? v[j][i] - mu1[TOK ? 0 : i] : v[j][i]) * rs1[TOK ? 0 : i], pw[j][TOK ? i : 0], pb[j][TOK ? i : 0]);
        ti.store(a.n, a.n_bs, b, t, v);
      }
      if (a.stats && ti.ch == 0) {
        const long bp = (long)a.B * a.P;
        float* sp = a.stats + (long)b * a.P + ti.pixel(t);
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (i >= NS - px) {
            sp[i] = mu0[i];
            sp[bp + i] = rs0[i];
            sp[2 * bp + i] = mu1[i];
            sp[3 * bp + i] = rs1[i];
          }
      }
    }
  }
}

// Backward.  Every operand once; the parameter gradients accumulate in the registers of the threads that hold the
// channel, over all of the worker's tiles, and are added up across lanes and waves once, at the end.  Tokens 4x4096x2048
// bf16 with both norms and a gate take 79 us (411 MB with the partial sums, 5.2 TB/s), planar 2x64x65536 fp32 32 us
// (169 MB, 5.2 TB/s), planar 2x512x256 fp32 6.8 us; the reduction of the partial sums behind it 3.4 to 7.5 us.
template <typename T, bool TOK, int L, int NV, int VEC, int NT, int MODE>
__global__ __launch_bounds__(TOK && L ? RN_LANE_T : RN_T) void rn_bwd_tile(const RnArgs a) {
  typedef Tile<T, TOK, L, NV, VEC, NT> Ti;
  typedef typename Ti::Vec Vec;
  constexpr int NS = Ti::NS, NP = Ti::NP;
  constexpr bool BR = MODE != RN_BWD_STREAM, IG = MODE == RN_BWD_IMAGE_GATE;
  constexpr int EW = NV * NP;                                  // channels of a thread
  // the next tile's operands are fetched ahead where the registers (256 per thread) have room for two tiles
  constexpr bool PF = !(BR && NV * VEC == 16 && (sizeof(T) == 4 || IG));
  __shared__ __attribute__((aligned(32))) float lds[Ti::RED];
  __shared__ float wsum[TOK && L ? RN_LANE_T / 64 * L * EW : 1];
  Ti ti(a, lds);
  int b0, b1, t0;
  ti.range(ti.worker(), b0, b1, t0);
  const int slab = t0, t1 = a.tiles;                           // (a worker behind the last image still writes its sums, zeros)
  float acc[RN_Q_N][NV][NP], img[2][NV][NP];                   // img: G1, G0 of the current image
#pragma unroll
  for (int q = 0; q < RN_Q_N; ++q)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < NP; ++i) acc[q][j][i] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < NP; ++i) img[0][j][i] = img[1][j][i] = 0.f;
  float pw[NV][NP], gw[NV][NP];
  const float inv = 1.0f / (float)a.C;
  const long bp = (long)a.B * a.P;
  // the operands of the next tile, and its statistics
  Vec dyn[NV], dnn[NV], yn[NV], fn[NV];
  float sn[4][NS];
  auto fetch = [&](int b, int t) {
    const unsigned st = ti.start(t);
    const float* sp = a.stats_in + (long)b * a.P + ti.pixel(t);
    if (a.pre) {
      ti.load(Ti::image(a.dn, a.dn_bs, b), st, dnn);
      ti.load(Ti::image(a.y_in, a.yi_bs, b), st, yn);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        sn[2][i] = sp[2 * bp + i];
        sn[3][i] = sp[3 * bp + i];
      }
    }
    if (a.dy) ti.load(Ti::image(a.dy, a.dy_bs, b), st, dyn);
    if (BR) {
      ti.load(Ti::image(a.f, a.f_bs, b), st, fn);
      if (a.post) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          sn[0][i] = sp[i];
          sn[1][i] = sp[bp + i];
        }
      }
    }
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) dyn[j].v = dnn[j].v = yn[j].v = fn[j].v = typename Vec::V(0);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    sn[0][i] = sn[2][i] = sn[3][i] = 0.f;
    sn[1][i] = 1.f;
  }
  if (PF && b0 < b1) fetch(b0, t0);
  ti.params(a.pre ? a.pre_w : nullptr, 0.f, pw);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < NP; ++i) gw[j][i] = 0.f;
  bool have_gw = false;
  for (int b = b0; b < b1; ++b) {
    if (BR && (!have_gw || IG)) {
      have_gw = true;
      ti.params(a.post ? a.post_w : nullptr, 1.f, gw);
      float g[NV][NP];
      ti.params(a.gate_kind ? a.gate + (IG ? (long)b * a.C : 0) : nullptr, 1.f, g);
      // 0 for a channel that is not the thread's own: it then adds nothing to the sums
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < NP; ++i) gw[j][i] = ti.exists(j, i) ? gw[j][i] * g[j][i] : 0.f;
    }
    const float s = a.scale ? a.scale[b] : 1.0f;
    for (int t = t0; t < t1; t += a.S) {
      if (!PF) fetch(b, t);
      Vec dy[NV], dn[NV], yv[NV], fv[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        dy[j] = dyn[j];
        dn[j] = dnn[j];
        yv[j] = yn[j];
        fv[j] = fn[j];
      }
      float mu0[NS], rs0[NS], mu1[NS], rs1[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        mu0[i] = sn[0][i];
        rs0[i] = sn[1][i];
        mu1[i] = sn[2][i];
        rs1[i] = sn[3][i];
      }
      const int bn = t + a.S < t1 ? b : b + 1, tn = t + a.S < t1 ? t + a.S : t0;
      if (PF && bn < b1) fetch(bn, tn);
      const int px = ti.own_pixels(t);
      // a pixel that is not the vector's own is all zeros below, whatever stands there: it adds nothing to any sum
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (!TOK && i < VEC - px) mu0[i] = rs0[i] = mu1[i] = rs1[i] = 0.f;
      float d[NV][VEC];                                        // dyt
      if (a.pre) {
        float m[2 * NS];
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) m[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int q = TOK ? 0 : i, c = TOK ? i : 0;
            const bool own = ti.mine(j, i, px);
            const float o = own ? dn[j].at(i) : 0.f, yo = own ? yv[j].at(i) : 0.f, g = o * pw[j][c];
            const float vh = (a.pre == 1 ? yo - mu1[q] : yo) * rs1[q];
            m[q] += g;
            m[NS + q] = fmaf(g, vh, m[NS + q]);
            acc[RN_Q_PRE_W][j][c] = fmaf(o, vh, acc[RN_Q_PRE_W][j][c]);
            acc[RN_Q_PRE_B][j][c] += o;
          }
        ti.template reduce<2 * NS>(m);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          m[i] = a.pre == 1 ? m[i] * inv : 0.f;
          m[NS + i] *= inv;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int q = TOK ? 0 : i, c = TOK ? i : 0;
            const float cent = (yv[j].at(i) - mu1[q]) * rs1[q];
            d[j][i] = fmaf(rs1[q], dn[j].at(i) * pw[j][c] - m[q] - cent * m[NS + q], dy[j].at(i));
          }
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[j][i] = dy[j].at(i);
      }
      if (a.dx) ti.store(a.dx, a.dx_bs, b, t, d);
      if (!BR) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) d[j][i] *= s;
      } else {
        float m[2 * NS];
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) m[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int q = TOK ? 0 : i, c = TOK ? i : 0;
            const bool own = ti.mine(j, i, px);
            const float sd = own ? d[j][i] * s : 0.f, fo = own ? fv[j].at(i) : 0.f;
            const float vh = (a.post == 1 ? fo - mu0[q] : fo) * rs0[q];
            img[0][j][c] = fmaf(sd, vh, img[0][j][c]);
            img[1][j][c] += sd;
            d[j][i] = sd * gw[j][c];
            m[q] += d[j][i];
            m[NS + q] = fmaf(d[j][i], vh, m[NS + q]);
          }
        if (a.post) {
          ti.template reduce<2 * NS>(m);
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            m[i] = a.post == 1 ? m[i] * inv : 0.f;
            m[NS + i] *= inv;
          }
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const int q = TOK ? 0 : i;
              d[j][i] = rs0[q] * (d[j][i] - m[q] - (fv[j].at(i) - mu0[q]) * rs0[q] * m[NS + q]);
            }
        }
      }
      ti.store(a.df, a.df_bs, b, t, d);
    }
    if (IG) {
      // the image is done: its gate's gradient, and its share of the norm's parameters
      float w0[NV][NP], bb[NV][NP], g[NV][NP];
      ti.params(a.post ? a.post_w : nullptr, 1.f, w0);
      ti.params(a.post == 1 ? a.post_b : nullptr, 0.f, bb);
      ti.params(a.gate + (long)b * a.C, 0.f, g);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float g1 = img[0][j][i], g0 = img[1][j][i];
          if (!TOK) {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) {
              g1 += __shfl_xor(g1, o);
              g0 += __shfl_xor(g0, o);
            }
          }
          acc[RN_Q_G1][j][i] = fmaf(img[0][j][i], g[j][i], acc[RN_Q_G1][j][i]);
          acc[RN_Q_G0][j][i] = fmaf(img[1][j][i], g[j][i], acc[RN_Q_G0][j][i]);
          img[0][j][i] = img[1][j][i] = 0.f;
          const float dg = fmaf(g1, w0[j][i], g0 * bb[j][i]);
          if (ti.exists(j, i) && (TOK || ti.pl == 0)) {
            const int c = ti.channel(j) + i;
            if (a.S > 1) {
              if (a.part_gate) a.part_gate[((long)b * a.S + slab) * a.C + c] = dg;
            } else if (a.dgate) {
              a.dgate[(long)b * a.C + c] = a.accumulate ? a.dgate[(long)b * a.C + c] + dg : dg;
            }
          }
        }
    }
  }
  if (!a.part) return;
  // one row of partial sums per workgroup, for the quantities that are wanted
#pragma unroll
  for (int q = 0; q < RN_Q_N; ++q) {
    if ((!BR && q < RN_Q_PRE_W) || !(a.wanted >> q & 1)) continue;
    float* out = a.part + ((long)q * a.part_rows + blockIdx.x) * a.C;
    if (TOK && L) {
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float v = BR && !IG && q < RN_Q_PRE_W ? img[q][j][i] : acc[q][j][i];
#pragma unroll
          for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o);
          if (lane < L) wsum[(wave * L + lane) * EW + j * NP + i] = v;
        }
      __syncthreads();
      for (int k = threadIdx.x; k < L * EW; k += blockDim.x) {
        const int l = k / EW, e = k % EW, c0 = ((e / NP) * L + l) * VEC, c = min(c0, a.C - VEC) + e % NP;
        float v = 0.f;
        for (int w = 0; w < waves; ++w) v += wsum[(w * L + l) * EW + e];
        if (c >= c0) out[c] = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float v = BR && !IG && q < RN_Q_PRE_W ? img[q][j][i] : acc[q][j][i];
          if (!TOK) {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
          }
          if (ti.exists(j, i) && (TOK || ti.pl == 0)) out[ti.channel(j) + i] = v;
        }
    }
  }
}

// ---- any number of channels -------------------------------------------------------------------------------------------
// One workgroup per token (tokens layout, 256 threads along the channels) or per 64 pixels (planar, four waves along
// the channels); nothing is kept between the passes over the channels, each reads its operands again.  That costs: where the
// register form fits it takes 196 us for tokens 8x4096x4096 bf16, this one 1306 us; planar 2x32x65536 fp32 14 and 31 us;
// backward of tokens 4x4096x2048 bf16 83 and 544 us.
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
    T* dx = a.dx ? static_cast<T*>(a.dx) + b * a.dx_bs + o : nullptr;
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
        if (dx) Elem<T>::st(dx + c * a.cs, d);
        Elem<T>::st(df + c * a.cs, du);
      }
  }
}

// The parameter gradients of the sweep form: one pass more over the operands, a workgroup per 64 channels and worker
// (tokens: lanes along the channels, waves along the rows; planar: a wave per channel, lanes along the pixels).
template <typename T, bool TOK>
__global__ __launch_bounds__(256) void rn_bwd_params_sweep(const RnArgs a) {
  __shared__ float red[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int worker = blockIdx.y;
  const int b0 = a.S > 1 ? worker / a.S : worker * a.ipw, b1 = (int)min((long)a.B, (long)b0 + a.ipw);   // (S > 1: ipw is 1)
  const int slab = a.S > 1 ? worker % a.S : 0;
  const long per = ((long)a.P + a.S - 1) / a.S, p0 = min((long)a.P, slab * per), p1 = min((long)a.P, p0 + per);
  const long bp = (long)a.B * a.P;
  const int c = blockIdx.x * (TOK ? 64 : 4) + (TOK ? lane : wave);
  const bool on = c < a.C;
  const int cc = on ? c : 0;
  float acc[RN_Q_N] = {0.f, 0.f, 0.f, 0.f};
  // per-channel sums across the threads that share the channel
  auto total = [&](float v) {
    if (!TOK) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
      return v;
    }
    __syncthreads();
    red[tid] = v;
    __syncthreads();
    return (red[lane] + red[64 + lane]) + (red[128 + lane] + red[192 + lane]);
  };
  const bool writer = on && (TOK ? wave == 0 : lane == 0);
  const bool branch = a.post || a.gate_kind;
  for (int b = b0; b < b1; ++b) {
    const float s = a.scale ? a.scale[b] : 1.0f;
    const float w1 = a.pre ? a.pre_w[cc] : 0.f;
    float g1 = 0.f, g0 = 0.f;
    for (long p = p0 + (TOK ? wave : lane); p < p1; p += TOK ? 4 : 64) {
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
        acc[RN_Q_PRE_W] = fmaf(dnv, (a.pre == 1 ? yv - r.mu1 : yv) * r.rs1, acc[RN_Q_PRE_W]);
        acc[RN_Q_PRE_B] += dnv;
      }
      if (!branch) continue;
      const float d = rn_dyt(a, r, a.dy ? Elem<T>::ld(static_cast<const T*>(a.dy) + b * a.dy_bs + o) : 0.f, dnv, yv, w1) * s;
      float u = Elem<T>::ld(static_cast<const T*>(a.f) + b * a.f_bs + o);
      if (a.post) u = (a.post == 1 ? u - a.stats_in[at] : u) * a.stats_in[bp + at];
      g1 = fmaf(d, u, g1);
      g0 += d;
    }
    if (branch && a.gate_kind == 2) {
      const float w0 = a.post ? a.post_w[cc] : 1.f, bb = a.post == 1 && a.post_b ? a.post_b[cc] : 0.f;
      const float gt = a.gate[(long)b * a.C + cc];
      const float dg = fmaf(total(g1), w0, total(g0) * bb);
      if (writer) {
        if (a.S > 1) {
          if (a.part_gate) a.part_gate[((long)b * a.S + slab) * a.C + c] = dg;
        } else if (a.dgate) {
          a.dgate[(long)b * a.C + c] = a.accumulate ? a.dgate[(long)b * a.C + c] + dg : dg;
        }
      }
      g1 *= gt;
      g0 *= gt;
    }
    acc[RN_Q_G1] += g1;
    acc[RN_Q_G0] += g0;
  }
#pragma unroll
  for (int q = 0; q < RN_Q_N; ++q) {
    const float v = total(acc[q]);
    if (writer) a.part[((long)q * a.part_rows + worker) * a.C + c] = v;
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
// Vectors: 16 bytes of channels per thread in the token layout, four pixels in the planar one.
template <typename T> constexpr int rn_vec(bool tok) { return tok ? 16 / (int)sizeof(T) : 4; }
unsigned sweep_blocks(bool tok, int B, int P) {
  const long tiles = (tok ? (long)P : ((long)P + 63) / 64) * B;
  return (unsigned)std::min<long>(tiles, 1 << 16);
}

// A form that choose_form gives and no kernel is built for would leave the outputs unwritten: an error instead.
[[noreturn]] inline void no_kernel(const RnForm& f) {
  set_error("residual_norm: no %s kernel of %d lanes and %d vectors", f.tok ? "token" : "planar", f.lanes, f.nv);
  throw Failure{JIRF_EINVAL};
}

#define RN_FWD_NT(TOK, L, NV, NT)                                                                                         \
  hipLaunchKernelGGL((rn_fwd_tile<T, TOK, L, NV, rn_vec<T>(TOK), NT>), dim3(f.blocks), dim3(f.threads), 0, s, a)
#define RN_FWD(TOK, L, NV) RN_FWD_NT(TOK, L, NV, 0)
template <typename T>
void launch_fwd(const RnArgs& a, const RnForm& f, hipStream_t s) {
  constexpr int E8 = 8 / rn_vec<T>(true);       // vectors for eight channels per thread
  if (f.lanes < 0) {
    if (f.tok) hipLaunchKernelGGL((rn_fwd_sweep<T, true>), dim3(sweep_blocks(true, a.B, a.P)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rn_fwd_sweep<T, false>), dim3(sweep_blocks(false, a.B, a.P)), dim3(256), 0, s, a);
  } else if (f.tok) {
    switch (f.lanes) {
      case 4: RN_FWD(true, 4, E8); break;
      case 8: RN_FWD(true, 8, E8); break;
      case 16: RN_FWD(true, 16, E8); break;
      case 32: RN_FWD(true, 32, E8); break;
      case 64: RN_FWD(true, 64, E8); break;
      case 0:
        if (f.nv == E8) {
          if (f.stream == 2) RN_FWD_NT(true, 0, E8, 2);
          else if (f.stream) RN_FWD_NT(true, 0, E8, 1);
          else RN_FWD(true, 0, E8);
        } else {
          if (f.stream == 2) RN_FWD_NT(true, 0, 2 * E8, 2);
          else if (f.stream) RN_FWD_NT(true, 0, 2 * E8, 1);
          else RN_FWD(true, 0, 2 * E8);
        }
        break;
      default: no_kernel(f);
    }
  } else {
    if constexpr (sizeof(T) == 4) {
      if (f.nv == 8) {
        switch (f.lanes) {
          case 2: RN_FWD(false, 2, 8); break;
          case 4: RN_FWD(false, 4, 8); break;
          case 8: RN_FWD(false, 8, 8); break;
          default: no_kernel(f);
        }
        return;
      }
    }
    switch (f.lanes) {
      case 2:
        if constexpr (sizeof(T) == 2) RN_FWD(false, 2, 4);
        else no_kernel(f);
        break;
      case 4: RN_FWD(false, 4, 4); break;
      case 8: RN_FWD(false, 8, 4); break;
      case 16: RN_FWD(false, 16, 4); break;
      case 32: RN_FWD(false, 32, 4); break;
      default: no_kernel(f);
    }
  }
}
#undef RN_FWD
#undef RN_FWD_NT

#define RN_BWD_NT(TOK, L, NV, NT)                                                                                         \
  hipLaunchKernelGGL((rn_bwd_tile<T, TOK, L, NV, rn_vec<T>(TOK), NT, MODE>), dim3(f.blocks), dim3(f.threads), 0, s, a)
#define RN_BWD(TOK, L, NV) RN_BWD_NT(TOK, L, NV, 0)
template <typename T, int MODE>
void launch_bwd_tile(const RnArgs& a, const RnForm& f, hipStream_t s) {
  constexpr int E8 = 8 / rn_vec<T>(true);
  if (f.tok) {
    switch (f.lanes) {
      case 4: RN_BWD(true, 4, E8); break;
      case 8: RN_BWD(true, 8, E8); break;
      case 16: RN_BWD(true, 16, E8); break;
      case 32: RN_BWD(true, 32, E8); break;
      case 64: RN_BWD(true, 64, E8); break;
      case 0:
        if (f.nv == E8 && f.stream) RN_BWD_NT(true, 0, E8, 1);
        else if (f.nv == E8) RN_BWD(true, 0, E8);
        else if (f.stream) RN_BWD_NT(true, 0, 2 * E8, 1);
        else RN_BWD(true, 0, 2 * E8);
        break;
      default: no_kernel(f);
    }
  } else {
    switch (f.lanes) {
      case 2: RN_BWD(false, 2, 4); break;
      case 4: RN_BWD(false, 4, 4); break;
      case 8: RN_BWD(false, 8, 4); break;
      case 16: RN_BWD(false, 16, 4); break;
      case 32: RN_BWD(false, 32, 4); break;
      default: no_kernel(f);
    }
  }
}
#undef RN_BWD
#undef RN_BWD_NT
template <typename T>
void launch_bwd(const RnArgs& a, const RnForm& f, int mode, bool params, hipStream_t s) {
  if (f.lanes < 0) {
    const dim3 grid(sweep_blocks(f.tok, a.B, a.P));
    const dim3 pgrid((unsigned)((a.C + (f.tok ? 63 : 3)) / (f.tok ? 64 : 4)), (unsigned)a.part_rows);
    if (f.tok) {
      hipLaunchKernelGGL((rn_bwd_sweep<T, true>), grid, dim3(256), 0, s, a);
      if (params) hipLaunchKernelGGL((rn_bwd_params_sweep<T, true>), pgrid, dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((rn_bwd_sweep<T, false>), grid, dim3(256), 0, s, a);
      if (params) hipLaunchKernelGGL((rn_bwd_params_sweep<T, false>), pgrid, dim3(256), 0, s, a);
    }
  } else if (mode == RN_BWD_STREAM) {
    launch_bwd_tile<T, RN_BWD_STREAM>(a, f, s);
  } else if (mode == RN_BWD_BRANCH) {
    launch_bwd_tile<T, RN_BWD_BRANCH>(a, f, s);
  } else {
    launch_bwd_tile<T, RN_BWD_IMAGE_GATE>(a, f, s);
  }
}

}  // namespace
}  // namespace jirf
#endif  // JIRF_RN_KERNELS
