// Rotary positions over several axes, alone and behind a per-head RMS norm, forward and backward
// (include/turtle_token.h).
//
//   z = x r w, r = 1 / sqrt(mean(x^2) + eps)          (norm of a (token, head) row over its D channels)
//   y = R z: channel pair i of the row turns by pos[axis_i] f_i
//   backward: dz = R^T dy, g = dz w, dx = r (g - x r^2 mean(g x)), dw = sum over rows of dz x r
//
// Bound: HBM - x in, y out (backward: x, dy in, dx out) and nothing in between. A row of D channels sits on
// D / 8 lanes (rounded up to a power of two), 8 channels a lane, so the norm's sums are a few DPP steps. A
// thread keeps ONE token and channel chunk and walks over the heads of q and k: the angles (4 pairs a lane) are
// computed once for all of them.
//
// Measured: 32640 tokens, 8 + 8 heads of 64 channels, bf16: 34 us (3.9 TB/s; a large copy reaches 4.9); 40960 tokens,
// forward 42 us, backward with both gains' gradients 57 + 4 us (4.4 TB/s).
//
// Angles: f_i is a 64-bit fixed-point number of revolutions per position, so pos * f_i wraps exactly: what is lost is
// |pos| 2^-65 revolutions of f_i's rounding, and position 10^6 is as precise as position 0 (fp32 products would be off by
// 0.06 rad there).
#include "common.h"
#include "../../include/turtle_token.h"

#include <algorithm>
#include <type_traits>

namespace turtle {
namespace {

typedef turtle_token_side Side;
typedef turtle_token_axes Axes;

constexpr int NTHR = 256;
constexpr int U = 2;              // rows of each tensor a thread has in flight
constexpr int MAXB = 1024;        // blocks of the backward: its dw partials are one row of 2 D floats a block

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// 8 elements as loaded: unpacked when they are used, so that rows in flight take few registers
template <typename T> struct Raw {
  uint4 q;
  TURTLE_DEV void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
  TURTLE_DEV void zero() { q = make_uint4(0, 0, 0, 0); }
  TURTLE_DEV void get(float (&v)[8]) const {
    if constexpr (std::is_same<T, bf16>::value) {
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
      const f16x8 x = __builtin_bit_cast(f16x8, q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    }
  }
};
template <> struct Raw<float> {
  float4 a, b;
  TURTLE_DEV void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
  TURTLE_DEV void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  TURTLE_DEV void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};
TURTLE_DEV void st8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
TURTLE_DEV void st8(bf16* p, const float (&v)[8]) {
  bf16x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
  *reinterpret_cast<bf16x8*>(p) = o;
}
TURTLE_DEV void st8(f16* p, const float (&v)[8]) {
  f16x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (f16)v[i];
  *reinterpret_cast<f16x8*>(p) = o;
}

// sine and cosine of hi / 2^32 revolutions. 16-bit results: the hardware functions (they take revolutions; their
// error is far under the results' rounding). fp32: the nearest quarter turn is split off exactly, the rest, at
// most pi / 4, goes through the Taylor polynomials up to x^9 and x^10 (truncation under 4e-9).
template <typename T>
TURTLE_DEV void sincos_rev(uint32_t hi, float& s, float& c) {
  if constexpr (sizeof(T) == 2) {
    const float t = (float)(int32_t)hi * 2.3283064365386963e-10f;
    s = __builtin_amdgcn_sinf(t);
    c = __builtin_amdgcn_cosf(t);
  } else {
    const uint32_t q = (hi + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(hi - (q << 30)) * (6.283185307179586f * 2.3283064365386963e-10f), u = x * x;
    const float sx = x * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
    const float cx = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const float a = (q & 1) ? cx : sx, b = (q & 1) ? sx : cx;
    s = (q & 2) ? -a : a;
    c = ((q + 1) & 2) ? -b : b;
  }
}

// sum over aligned groups of 2^LB lanes (LB <= 4), in every lane of the group
template <int LB>
TURTLE_DEV float row_sum(float v) {
  if constexpr (LB >= 1) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));    // lane ^ 1
  if constexpr (LB >= 2) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true));    // lane ^ 2
  if constexpr (LB >= 3) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, true));   // mirror of 8
  if constexpr (LB >= 4) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, true));   // mirror of 16
  return v;
}

// 1 / sqrt(x): the hardware's (one ulp or so); fp32 with a Newton step, but 0 of infinity (a row whose squares pass fp32)
template <typename T>
TURTLE_DEV float rsqrt_of(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  if constexpr (sizeof(T) == 2) return r;
  else return x < INFINITY ? r * fmaf(-0.5f * x * r, r, 1.5f) : r;
}

struct RopeArgs {
  Side s[2];
  Axes ax;
  const void* pos;
  int64_t pos_b, S, B;
  int D, hs;                 // hs: threads (a power of two) that share a token's heads
  int pos64, whole;          // whole: every channel is rotated
  float eps;
  float* part;               // backward: [gridDim.x][2][D] or NULL
};

// a lane's place: its chunk of 8 channels, its share of the heads, its token within the block's step
struct Place {
  int c, h0, tok, step;
  bool on;
  template <int LB>
  TURTLE_DEV static Place of(const RopeArgs& a) {
    Place p;
    const int slot = threadIdx.x >> LB;
    p.c = (threadIdx.x & ((1 << LB) - 1)) * 8;
    p.on = p.c < a.D;
    p.h0 = slot & (a.hs - 1);
    p.tok = slot / a.hs;
    p.step = (NTHR >> LB) / a.hs;
    return p;
  }
};

struct Turn {
  uint64_t f[4];
  int ax[4];
  bool rot[4];
  float s[4], c[4];
  TURTLE_DEV void init(const Axes& t, int c0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = (c0 >> 1) + i;
      rot[i] = p < t.npair;
      f[i] = rot[i] ? t.freq[p] : 0;
      ax[i] = rot[i] ? t.axis[p] : 0;
    }
  }
  template <typename T>
  TURTLE_DEV void at(const RopeArgs& a, int64_t b, int64_t t) {
    const int64_t o = b * a.pos_b + t * a.ax.naxis;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[o + ax[i]] : (int64_t)reinterpret_cast<const int32_t*>(a.pos)[o + ax[i]];
      sincos_rev<T>((uint32_t)(((uint64_t)p * f[i]) >> 32), s[i], c[i]);
    }
  }
  // channels that are not rotated pass unchanged, whatever they hold. INV: by the angle's negative
  template <bool INV>
  TURTLE_DEV void apply(float (&v)[8], bool whole) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = v[2 * i], x1 = v[2 * i + 1], sn = INV ? -s[i] : s[i];
      const float y0 = fmaf(x0, c[i], -x1 * sn), y1 = fmaf(x0, sn, x1 * c[i]);
      v[2 * i] = whole || rot[i] ? y0 : x0;
      v[2 * i + 1] = whole || rot[i] ? y1 : x1;
    }
  }
};

template <typename T, bool NORM, bool INV, int LB>
__global__ __launch_bounds__(NTHR) void rope_kernel(RopeArgs a) {
  const Place p = Place::of<LB>(a);
  const int H = max(a.s[0].H, a.s[1].H);
  const bool whole = a.whole;
  Turn tn;
  tn.init(a.ax, p.c);
  float w[2][8];
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] = (p.on && a.s[i].w) ? a.s[i].w[p.c + e] : 1.f;
  }
  const float invD = 1.f / (float)a.D;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y)
  for (int64_t t = (int64_t)blockIdx.x * p.step + p.tok; t < a.S; t += (int64_t)gridDim.x * p.step) {
    for (int h0 = p.h0; h0 < H; h0 += U * a.hs) {
      Raw<T> x[2][U];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.hs;
          x[k][u].zero();
          if (h < a.s[k].H && p.on) x[k][u].load(reinterpret_cast<const T*>(a.s[k].x) + b * a.s[k].sb + t * a.s[k].ss + h * a.s[k].sh + p.c);
        }
      if (h0 == p.h0) tn.at<T>(a, b, t);      // the angles while the first rows are on their way
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.hs;
          float v[8];
          x[k][u].get(v);
          if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
            const float r = rsqrt_of<T>(fmaf(row_sum<LB>(ss), invD, a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= r * w[k][e];
          }
          tn.apply<INV>(v, whole);
          if (h < a.s[k].H && p.on) st8(reinterpret_cast<T*>(a.s[k].y) + ((b * a.S + t) * a.s[k].H + h) * a.D + p.c, v);
        }
    }
  }
}

template <typename T, int LB>
__global__ __launch_bounds__(NTHR) void norm_rope_bwd_kernel(RopeArgs a) {
  const Place p = Place::of<LB>(a);
  const int H = max(a.s[0].H, a.s[1].H);
  const bool whole = a.whole;
  Turn tn;
  tn.init(a.ax, p.c);
  float w[2][8], dw[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) { w[i][e] = (p.on && a.s[i].w) ? a.s[i].w[p.c + e] : 1.f; dw[i][e] = 0.f; }
  const float invD = 1.f / (float)a.D;
  for (int64_t b = blockIdx.y; b < a.B; b += gridDim.y)
  for (int64_t t = (int64_t)blockIdx.x * p.step + p.tok; t < a.S; t += (int64_t)gridDim.x * p.step) {
    for (int h0 = p.h0; h0 < H; h0 += U * a.hs) {
      Raw<T> rx[2][U], rg[2][U];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.hs;
          rx[k][u].zero();
          rg[k][u].zero();
          if (h < a.s[k].H && p.on) {
            rx[k][u].load(reinterpret_cast<const T*>(a.s[k].x) + b * a.s[k].sb + t * a.s[k].ss + h * a.s[k].sh + p.c);
            rg[k][u].load(reinterpret_cast<const T*>(a.s[k].dy) + b * a.s[k].gb + t * a.s[k].gs + h * a.s[k].gh + p.c);
          }
        }
      if (h0 == p.h0) tn.at<T>(a, b, t);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * a.hs;
          float x[8], g[8];
          rx[k][u].get(x);
          rg[k][u].get(g);
          tn.apply<true>(g, whole);
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
          const float r = rsqrt_of<T>(fmaf(row_sum<LB>(ss), invD, a.eps));
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] *= r;
            dw[k][e] = fmaf(g[e], x[e], dw[k][e]);      // rows that are not there are zero
            g[e] *= w[k][e];
            dot = fmaf(g[e], x[e], dot);
          }
          const float m = row_sum<LB>(dot) * invD;
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = r * fmaf(-x[e], m, g[e]);
          if (h < a.s[k].H && p.on) st8(reinterpret_cast<T*>(a.s[k].y) + ((b * a.S + t) * a.s[k].H + h) * a.D + p.c, g);
        }
    }
  }
  if (!a.part) return;
  // the block's dw: over its slots in a fixed order
  __shared__ float red[NTHR * 8];
  for (int k = 0; k < 2; ++k) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = dw[k][e];
    __syncthreads();
    if ((int)threadIdx.x < a.D) {
      float s = 0.f;
      for (int i = 0; i < (NTHR >> LB); ++i) s += red[(i << LB) * 8 + threadIdx.x];
      a.part[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + k) * a.D + threadIdx.x] = s;
    }
  }
}

// dw[c] = sum over the blocks' partials: 16 of the 2 D columns a block, 4 a thread, 64 threads a column group
__global__ __launch_bounds__(NTHR) void dw_sum_kernel(const float* __restrict__ part, float* __restrict__ dw, int nblk, int cols) {
  __shared__ float4 red[NTHR];
  const int col = blockIdx.x * 16 + (threadIdx.x & 3) * 4, r0 = threadIdx.x >> 2;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int r = r0; r < nblk; r += 64) {
    const float4 x = *reinterpret_cast<const float4*>(part + (int64_t)r * cols + col);
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 16) {
    float t = 0.f;
    for (int i = 0; i < 64; ++i) t += reinterpret_cast<const float*>(&red[i * 4])[threadIdx.x];
    dw[blockIdx.x * 16 + threadIdx.x] = t;
  }
}

bool side_ok(const Side* s, int D, int es, bool bwd) {
  auto al = [&](int64_t st) { return (st * es) % 16 == 0; };
  if (!s->x || !s->y || s->H <= 0 || ((uintptr_t)s->x | (uintptr_t)s->y) % 16 || !al(s->sb) || !al(s->ss) || !al(s->sh)) return false;
  return !bwd || (s->dy && (uintptr_t)s->dy % 16 == 0 && al(s->gb) && al(s->gs) && al(s->gh));
}

// channel lanes of a row: log2 of D / 8 rounded up to a power of two
int lane_bits(int D) { int lb = 0; while ((8 << lb) < D) ++lb; return lb; }

bool fill(RopeArgs& r, const Side* a, const Side* b, const Axes* axes, const void* pos, int64_t pos_b, int pos64, int64_t B, int64_t S,
          int D, int dtype, bool bwd) {
  if (!a || !axes || !pos || B <= 0 || S <= 0 || D <= 0 || D % 8 || D > 128 || dtype < 0 || dtype > 2) return false;
  const int es = dtype == 0 ? 4 : 2;
  if (!side_ok(a, D, es, bwd) || (b && b->x && !side_ok(b, D, es, bwd))) return false;
  if (axes->npair < 0 || 2 * axes->npair > D || axes->naxis < 1 || axes->naxis > 4) return false;
  for (int i = 0; i < axes->npair; ++i)
    if (axes->axis[i] >= axes->naxis) return false;
  r = RopeArgs{};
  r.s[0] = *a;
  if (b && b->x) r.s[1] = *b;
  r.ax = *axes;
  r.pos = pos; r.pos_b = pos_b; r.pos64 = pos64;
  r.S = S; r.B = B; r.D = D;
  r.whole = 2 * axes->npair == D;
  // heads dealt so that a thread has about U rows of each tensor: they share its angles and are in flight together
  const int slots = NTHR >> lane_bits(D), H = std::max(r.s[0].H, r.s[1].H);
  int hs = 1;
  while (hs < slots && hs * U < H) hs *= 2;
  r.hs = hs;
  return true;
}

// blocks (x: tokens, y: sequences), at most `most` of them
dim3 blocks_for(const RopeArgs& r, int64_t most) {
  const int64_t step = (NTHR >> lane_bits(r.D)) / r.hs, y = std::min<int64_t>({r.B, most, 1 << 15});
  return dim3((unsigned)std::min<int64_t>((r.S + step - 1) / step, std::max<int64_t>(1, most / y)), (unsigned)y);
}

template <typename T, bool NORM, bool INV>
void launch_rope(const RopeArgs& r, hipStream_t st) {
  const dim3 g = blocks_for(r, 1 << 20);
  switch (lane_bits(r.D)) {
    case 0: rope_kernel<T, NORM, INV, 0><<<g, NTHR, 0, st>>>(r); break;
    case 1: rope_kernel<T, NORM, INV, 1><<<g, NTHR, 0, st>>>(r); break;
    case 2: rope_kernel<T, NORM, INV, 2><<<g, NTHR, 0, st>>>(r); break;
    case 3: rope_kernel<T, NORM, INV, 3><<<g, NTHR, 0, st>>>(r); break;
    default: rope_kernel<T, NORM, INV, 4><<<g, NTHR, 0, st>>>(r); break;
  }
}
template <typename T>
void launch_turn(const RopeArgs& r, bool inverse, hipStream_t st) {
  if (inverse) launch_rope<T, false, true>(r, st);
  else launch_rope<T, false, false>(r, st);
}
template <typename T>
void launch_bwd(const RopeArgs& r, dim3 g, hipStream_t st) {
  switch (lane_bits(r.D)) {
    case 0: norm_rope_bwd_kernel<T, 0><<<g, NTHR, 0, st>>>(r); break;
    case 1: norm_rope_bwd_kernel<T, 1><<<g, NTHR, 0, st>>>(r); break;
    case 2: norm_rope_bwd_kernel<T, 2><<<g, NTHR, 0, st>>>(r); break;
    case 3: norm_rope_bwd_kernel<T, 3><<<g, NTHR, 0, st>>>(r); break;
    default: norm_rope_bwd_kernel<T, 4><<<g, NTHR, 0, st>>>(r); break;
  }
}

}  // namespace
}  // namespace turtle

using namespace turtle;

extern "C" {

int turtle_token_rope(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes, const void* pos,
                      int64_t pos_b, int pos64, int64_t B, int64_t S, int D, int inverse, int dtype, void* stream) {
  RopeArgs r;
  if (!fill(r, a, b, axes, pos, pos_b, pos64, B, S, D, dtype, false)) return -1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) launch_turn<float>(r, inverse, st);
  else if (dtype == 1) launch_turn<bf16>(r, inverse, st);
  else launch_turn<f16>(r, inverse, st);
  return (int)hipGetLastError();
}

int turtle_token_norm_rope_fwd(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes,
                               const void* pos, int64_t pos_b, int pos64, int64_t B, int64_t S, int D, float eps, int dtype,
                               void* stream) {
  RopeArgs r;
  if (!fill(r, a, b, axes, pos, pos_b, pos64, B, S, D, dtype, false)) return -1;
  r.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) launch_rope<float, true, false>(r, st);
  else if (dtype == 1) launch_rope<bf16, true, false>(r, st);
  else launch_rope<f16, true, false>(r, st);
  return (int)hipGetLastError();
}

size_t turtle_token_norm_rope_workspace(int64_t tokens, int D) {
  if (tokens <= 0 || D <= 0) return 0;
  return (size_t)std::min<int64_t>(tokens, MAXB) * 2 * D * sizeof(float);
}

int turtle_token_norm_rope_bwd(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes,
                               const void* pos, int64_t pos_b, int pos64, int64_t B, int64_t S, int D, float eps, float* dw,
                               void* ws, size_t ws_bytes, int dtype, void* stream) {
  RopeArgs r;
  if (!fill(r, a, b, axes, pos, pos_b, pos64, B, S, D, dtype, true)) return -1;
  const dim3 g = blocks_for(r, dw ? MAXB : 1 << 20);
  const int nblk = (int)(g.x * g.y);
  if (dw && (!ws || (uintptr_t)ws % 16 || ws_bytes < (size_t)nblk * 2 * D * sizeof(float))) return -1;
  r.eps = eps;
  r.part = dw ? (float*)ws : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) launch_bwd<float>(r, g, st);
  else if (dtype == 1) launch_bwd<bf16>(r, g, st);
  else launch_bwd<f16>(r, g, st);
  if (dw) dw_sum_kernel<<<2 * D / 16, NTHR, 0, st>>>((const float*)ws, dw, nblk, 2 * D);
  return (int)hipGetLastError();
}

}  // extern "C"
