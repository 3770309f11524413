// Token attention, backward (token_attn.h holds the method and the shared parts): delta, then dk and dv by key tiles,
// then dq by row tiles. No atomics: every sum has a fixed order.
#include "token_attn.h"
#ifndef DKV_WAVES
#define DKV_WAVES (sizeof(T)==2 && DP==64 ? 2 : 1)
#endif
#ifndef DQ_WAVES
#define DQ_WAVES (sizeof(T)==2 && RW==1 ? 2 : 1)
#endif
#ifndef DKV_NS64
#define DKV_NS64 4
#endif
#ifndef DKV_NS128
#define DKV_NS128 4
#endif
#ifndef DQ_NS64
#define DQ_NS64 4
#endif
#ifndef DQ_NS128
#define DQ_NS128 (sizeof(T)==4?3:4)
#endif
#ifndef WKMAX
#define WKMAX 128
#endif

namespace turtle {
namespace {

__device__ const float g_row_pad[2] = {INFINITY, 0.f};   // softmax sum and delta of a row that is not there

// 64 lanes x 4 B -> LDS
TURTLE_DEV void dma4(const void* gp, uint32_t lds_wave_base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(gp), "s"(lds_wave_base) : "memory");
}

// delta [B][Hk][M] = do . (o + o_lo); 8 lanes a row, 16 bytes a lane and step
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(Args a, float* delta) {
  constexpr int V = 16 / sizeof(T);
  const int64_t u = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int64_t n = (int64_t)a.B * a.Sq * a.Hq;
  const int ln = threadIdx.x & 7;
  float s = 0.f;
  if (u < n) {
    const int64_t b = u / ((int64_t)a.Sq * a.Hq), j = u - b * a.Sq * a.Hq, i = j / a.Hq, hq = j - i * a.Hq;
    const T* g = reinterpret_cast<const T*>(a.dout) + b * a.gb + i * a.gs + hq * a.gh;
    const T* o = reinterpret_cast<const T*>(a.o) + u * a.D;
    const T* lo = a.olo ? reinterpret_cast<const T*>(a.olo) + u * a.D : nullptr;
    typedef T tv __attribute__((ext_vector_type(V)));
    for (int d = ln * V; d < a.D; d += 8 * V) {
      const tv x = *reinterpret_cast<const tv*>(g + d), y = *reinterpret_cast<const tv*>(o + d);
      tv z = {};
      if (lo) z = *reinterpret_cast<const tv*>(lo + d);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf((float)x[e], (float)y[e] + (float)z[e], s);
    }
    s += __shfl_xor(s, 1, 64); s += __shfl_xor(s, 2, 64); s += __shfl_xor(s, 4, 64);
    if (ln == 0) delta[((b * a.Hk + hq / a.G) * a.Sq + i) * a.G + hq % a.G] = s;
  }
}

// WK: for small grids - the block's NW waves own the same 32 keys and take the row tiles in turn, each with its own
// ring and no barriers, and join at the end
template <typename T, int DP, int NW, bool WK> struct Dkv {
  typedef Rows<T, DP> R;
  static constexpr int NT = NW * 64, LT = WK ? 64 : NT;
  static constexpr int BK = WK ? 32 : NW * 32;            // keys of a block
  static constexpr int BM = 32;                           // rows of a tile
  static constexpr int NS = WK ? 2 : (DP == 64 ? DKV_NS64 : DKV_NS128);
  static constexpr int TILE = BM * R::ROWB;
  static constexpr int INFO = 3 * BM * 4;                 // place, document, slope of each row
  static constexpr int SLOT = 2 * TILE + 64 * 4 + INFO;   // Q, dO, 32 softmax sums and 32 deltas
  static constexpr int JOIN = R::DT * 16 * 64 * 4;
  static constexpr int LDS = NS * SLOT * (WK ? NW : 1) > JOIN ? NS * SLOT * (WK ? NW : 1) : JOIN;
  static constexpr int NLD = R::template loads2<BM, LT>() + 1;
};

// sum of the waves' accumulators through LDS, in wave order; every wave gets it
template <int NW, int DT>
TURTLE_DEV void join_waves(f32x16 (&acc)[DT], float* sum, int wave, int lane) {
  __syncthreads();
  for (int w = 0; w < NW; ++w) {
    if (wave == w) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float* p = sum + (dt * 16 + r) * 64 + lane;
          *p = (w ? *p : 0.f) + acc[dt][r];
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = sum[(dt * 16 + r) * 64 + lane];
}

template <typename T, int DP, int NW, bool WK>
__global__ __launch_bounds__(NW * 64, DKV_WAVES) void attn_dkv_kernel(Args a) {
  typedef Dkv<T, DP, NW, WK> C;
  typedef Rows<T, DP> R;
  constexpr int BM = C::BM, DT = R::DT, KG = 1, NS = C::NS, STEP = WK ? NW : 1;
  // fp16: p times 2^10 as operand of dv (p of 10^4 keys would lose bits below the type's normal range)
  constexpr float POFF = std::is_same<T, f16>::value ? 10.f : 0.f, PS = std::is_same<T, f16>::value ? 1.f / 1024.f : 1.f;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int kt = item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int k0 = kt * C::BK, k1 = min(k0 + C::BK, a.Sk), off = a.Sk - a.Sq;
  const int kw = k0 + (WK ? 0 : wave * 32), kw1 = min(kw + 32, a.Sk);
  const int pre = a.prefix ? a.prefix[b] : 0;
  int key[KG], kdoc[KG];
  bool kon[KG];
  uint4 kf[KG][R::STEPS], vf[KG][R::STEPS];
#pragma unroll
  for (int w = 0; w < KG; ++w) {
    key[w] = kw + w * 32 + (lane & 31);
    kdoc[w] = (a.kdoc && key[w] < a.Sk) ? a.kdoc[(int64_t)b * a.Sk + key[w]] : 0;
    kon[w] = key[w] < a.Sk && kdoc[w] >= 0;
    R::frag(kon[w] ? reinterpret_cast<const T*>(a.k) + (int64_t)b * a.kb + (int64_t)key[w] * a.ks + (int64_t)hk * a.kh : nullptr, a.D, kf[w], lane);
    R::frag(kon[w] ? reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vb + (int64_t)key[w] * a.vs + (int64_t)hk * a.vh : nullptr, a.D, vf[w], lane);
  }

  // rows that may see a key of this block
  int mfirst = 0;
  if (a.causal && k0 >= pre) mfirst = max(0, k0 - off) * a.G;
  const int t1 = (a.M + BM - 1) / BM, t0 = min(t1, mfirst / BM);
  DocWalk dw;
  dw.init(nullptr, 0, make_int4(0, 0, 0, 0));
  if (a.qdoc) dw.init(a.qr + (int64_t)b * a.nqr, a.nqr, doc_range(a.kr + (int64_t)b * a.nkr, a.nkr, k0, k1));
  const float sl = (a.slopes && lane < a.G) ? a.slopes[hk * a.G + lane] * LOG2E : 0.f;
  const bool rules = a.causal || a.slopes || a.qdoc;

  const char* qbase = reinterpret_cast<const char*>(a.q) + ((int64_t)b * a.qb + (int64_t)hk * a.G * a.qh) * R::ES;
  const char* gbase = reinterpret_cast<const char*>(a.dout) + ((int64_t)b * a.gb + (int64_t)hk * a.G * a.gh) * R::ES;
  // where a tile holds whole tokens, its rows lie at the same offsets from its first one every time
  constexpr int NI = BM * R::CH / C::LT;
  const int ltid = WK ? lane : tid;
  char* ring = smem + (WK ? wave * NS * C::SLOT : 0);
  const bool plain = BM % a.G == 0 && a.D == DP;
  const int per = BM / a.G;
  int64_t qoff[NI], goff[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (i * C::LT + ltid) / R::CH, c = ((ltid % R::CH) ^ R::swz(r)) << 4, ti = r / a.G, g = r - ti * a.G;
    qoff[i] = ((int64_t)ti * a.qs + (int64_t)g * a.qh) * R::ES + c;
    goff[i] = ((int64_t)ti * a.gs + (int64_t)g * a.gh) * R::ES + c;
  }
  auto issue = [&](int t, char* dst) {
    if (rules && ltid < 64) {
      const int m = t * BM + (lane & 31), i = m / a.G, g = m - i * a.G;
      float s = 0.f;
      if (a.slopes) s = a.G <= 64 ? __shfl(sl, g, 64) : a.slopes[hk * a.G + g] * LOG2E;
      int d = 0;
      if (dw.mixed) d = m < a.M ? a.qdoc[(int64_t)b * a.Sq + i] : -1;
      int* info = reinterpret_cast<int*>(dst + 2 * C::TILE + 256);
      if (lane < BM) { info[lane] = i + off; info[BM + lane] = d; info[2 * BM + lane] = __float_as_int(s); }
    }
    const bool holes = dw.holes;
    if (plain && !holes && t * BM + BM <= a.M && (!a.causal || t * per + off >= 0 || pre > 0)) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t at = (uint32_t)(i * C::LT + (ltid & ~63)) * 16;
        dma16(qbase + qoff[i] + (int64_t)t * per * a.qs * R::ES, __builtin_amdgcn_readfirstlane(lds_addr(dst) + at));
        dma16(gbase + goff[i] + (int64_t)t * per * a.gs * R::ES, __builtin_amdgcn_readfirstlane(lds_addr(dst + C::TILE) + at));
      }
    } else
    R::template load2<BM, C::LT>(dst, dst + C::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
      const int m = t * BM + r, i = m / a.G, g = m - i * a.G;
      // rows that see nothing may hold anything: they are not read
      if (m >= a.M || (a.causal && i + off < 0 && pre <= 0) || (holes && a.qdoc[(int64_t)b * a.Sq + i] < 0)) return;
      p0 = qbase + ((int64_t)i * a.qs + (int64_t)g * a.qh) * R::ES;
      p1 = gbase + ((int64_t)i * a.gs + (int64_t)g * a.gh) * R::ES;
    });
    // every wave writes the same 64 values, so that all count the same number of loads
    const int m = t * BM + (lane & 31);
    const float* src = m < a.M ? (h ? a.delta : a.lse) + (int64_t)bh * a.M + m : g_row_pad + h;
    dma4(src, __builtin_amdgcn_readfirstlane(lds_addr(dst + 2 * C::TILE)));
  };

  f32x16 dk[KG][DT], dv[KG][DT];
#pragma unroll
  for (int w = 0; w < KG; ++w)
#pragma unroll
    for (int i = 0; i < DT; ++i) { dk[w][i] = zero16(); dv[w][i] = zero16(); }

  struct Tile { int t; bool mixed; } q[NS];
  auto next = [&](int t) { return dw.template next<BM, STEP>(t, t1, a.G, a.Sq, lane); };
  int slot = 0, fly = 0;
  auto fetch = [&](Tile& x, int t, int into) {
    x.t = next(t);
    x.mixed = dw.mixed;
    if (x.t < t1) { issue(x.t, ring + into * C::SLOT); ++fly; }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) fetch(q[i], i ? q[i - 1].t + STEP : (WK ? t0 + wave : t0), i);
  while (q[0].t < t1) {
    const int last = slot ? slot - 1 : NS - 1;
    if constexpr (WK) {
      fetch(q[NS - 1], q[NS - 2].t + STEP, last);
      vm_wait_tiles<C::NLD, NS - 1>(fly - 1);
    } else {
      vm_wait_tiles<C::NLD, NS - 2>(fly - 1);
      lds_barrier();
      fetch(q[NS - 1], q[NS - 2].t + STEP, last);
    }
    const char* qt = ring + slot * C::SLOT;
    const char* gt = qt + C::TILE;
    const float* in = reinterpret_cast<const float*>(qt + 2 * C::TILE);
    const int* info = reinterpret_cast<const int*>(qt + 2 * C::TILE + 256);
    const int t = q[0].t;
    const bool mixed = q[0].mixed;
    const int m0 = t * BM, m1 = min(m0 + BM, a.M);
    // causal: does any row of the tile see a key of this wave; do all see all of them
    const bool any = !a.causal || (m1 - 1) / a.G + off >= kw || kw < pre;
    if (any && kw < a.Sk) {
      f32x16 s[KG], dp[KG];
      R::template times<KG>(qt, 0, kf, s, lane);
      R::template times<KG>(gt, 0, vf, dp, lane);
      const bool caus = a.causal && m0 / a.G + off + 1 < kw1 && kw1 > pre;
      float mul = a.scale2;
      if (a.cap > 0.f) {
        tanh_all<T, KG>(s, a.icap);
        mul = a.cap2;
      }
      // dp -> (dp - delta) times the cap's slope
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 del = *reinterpret_cast<const float4*>(in + BM + 8 * c + 4 * h);
        const float de[4] = {del.x, del.y, del.z, del.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int w = 0; w < KG; ++w) {
            const int r = 4 * c + e;
            dp[w][r] = (dp[w][r] - de[e]) * PS;
            if (a.cap > 0.f) dp[w][r] *= fmaf(-s[w][r], s[w][r], 1.f);
          }
      }
      if (a.slopes) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int4 pos = *reinterpret_cast<const int4*>(info + 8 * c + 4 * h);
          const float4 slp = *reinterpret_cast<const float4*>(info + 2 * BM + 8 * c + 4 * h);
          const int po[4] = {pos.x, pos.y, pos.z, pos.w};
          const float sp[4] = {slp.x, slp.y, slp.z, slp.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int w = 0; w < KG; ++w) s[w][4 * c + e] = fmaf(-sp[e], fabsf((float)(po[e] - key[w])), s[w][4 * c + e] * mul);
        }
        mul = 1.f;
      }
      if (caus || mixed) {
        // the pairs that do not see each other: p = 0, and whatever dP holds there
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int4 pos = *reinterpret_cast<const int4*>(info + 8 * c + 4 * h), doc = *reinterpret_cast<const int4*>(info + BM + 8 * c + 4 * h);
          const int po[4] = {pos.x, pos.y, pos.z, pos.w}, dc[4] = {doc.x, doc.y, doc.z, doc.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int w = 0; w < KG; ++w) {
              bool vis = !caus || max(po[e], pre - 1) >= key[w];
              vis = vis && (!mixed || dc[e] == kdoc[w]);
              s[w][4 * c + e] = vis ? s[w][4 * c + e] * mul : -INFINITY;
              dp[w][4 * c + e] = vis ? dp[w][4 * c + e] : 0.f;
            }
        }
        mul = 1.f;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 lse = *reinterpret_cast<const float4*>(in + 8 * c + 4 * h);
        const float ls[4] = {lse.x, lse.y, lse.z, lse.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int w = 0; w < KG; ++w) {
            const int r = 4 * c + e;
            s[w][r] = __builtin_amdgcn_exp2f(fmaf(s[w][r], mul, POFF - ls[e]));
            dp[w][r] *= s[w][r];
          }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[KG][8], y[KG][8];
#pragma unroll
        for (int w = 0; w < KG; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) { x[w][e] = s[w][8 * u + e]; y[w][e] = dp[w][8 * u + e]; }
        R::template t_times<KG, false>(gt, u * 16, x, dv, lane);
        R::template t_times<KG, false>(qt, u * 16, y, dk, lane);
      }
    }
    if constexpr (WK) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    --fly;
    slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
    for (int i = 0; i + 1 < NS; ++i) q[i] = q[i + 1];
  }
  if constexpr (WK) {
    join_waves<NW>(dk[0], reinterpret_cast<float*>(smem), wave, lane);
    join_waves<NW>(dv[0], reinterpret_cast<float*>(smem), wave, lane);
  }
#pragma unroll
  for (int w = 0; w < KG; ++w) {
    if (key[w] >= a.Sk) continue;
    const int64_t oi = (((int64_t)b * a.Sk + key[w]) * a.Hk + hk) * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (WK && dt % NW != wave) continue;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d = dt * 32 + 8 * q4 + 4 * h;
        if (d >= a.D) continue;
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = kon[w] ? dk[w][dt][4 * q4 + e] * a.scale : 0.f;
          y[e] = kon[w] ? dv[w][dt][4 * q4 + e] * PS : 0.f;
        }
        R::put4(reinterpret_cast<T*>(a.dk) + oi + d, x);
        R::put4(reinterpret_cast<T*>(a.dv) + oi + d, y);
      }
    }
  }
}

template <typename T, int DP, int NW, int RW, bool WK> struct Dq {
  typedef Rows<T, DP> R;
  static constexpr int NT = NW * 64, LT = WK ? 64 : NT;
  static constexpr int WROWS = 32 * RW, BM = WK ? WROWS : NW * WROWS, BN = 32;
  static constexpr int NS = WK ? 2 : (DP == 64 ? DQ_NS64 : DQ_NS128);
  static constexpr int TILE = BN * R::ROWB, SLOT = 2 * TILE;
  static constexpr int JOIN = R::DT * 16 * 64 * 4;
  static constexpr int LDS = NS * SLOT * (WK ? NW : 1) > JOIN ? NS * SLOT * (WK ? NW : 1) : JOIN;
  static constexpr int NLD = R::template loads2<BN, LT>();
};

template <typename T, int DP, int NW, int RW, bool WK>
__global__ __launch_bounds__(NW * 64, DQ_WAVES) void attn_dq_kernel(Args a) {
  typedef Dq<T, DP, NW, RW, WK> C;
  typedef Rows<T, DP> R;
  constexpr int BN = C::BN, DT = R::DT, NS = C::NS, STEP = WK ? NW : 1;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int mt = a.mtiles - 1 - item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int off = a.Sk - a.Sq, m0 = mt * C::BM, m1 = min(m0 + C::BM, a.M);
  const int mw = m0 + (WK ? 0 : wave * C::WROWS), mw1 = min(mw + C::WROWS, a.M);
  const int pre = a.prefix ? a.prefix[b] : 0;
  int kend = a.Sk;
  if (a.causal) kend = min(a.Sk, max((m1 - 1) / a.G + off + 1, pre));
  const int t1 = (max(kend, 0) + BN - 1) / BN;
  DocWalk dw;
  dw.init(nullptr, 0, make_int4(0, 0, 0, 0));
  if (a.qdoc)
    dw.init(a.kr + (int64_t)b * a.nkr, a.nkr, doc_range(a.qr + (int64_t)b * a.nqr, a.nqr, m0 / a.G, (m1 - 1) / a.G + 1));
  const int whole = a.causal ? max(mw / a.G + off + 1, pre) : 0x7fffffff;
  const int some = mw1 <= mw ? 0 : (a.causal ? max((mw1 - 1) / a.G + off + 1, pre) : 0x7fffffff);

  int mrow[RW];
  Row row[RW];
  float lse[RW], delta[RW];
  uint4 qf[RW][R::STEPS], gf[RW][R::STEPS];
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    mrow[w] = mw + w * 32 + (lane & 31);
    row[w] = row_of(a, b, hk, mrow[w], off, a.Sq);
    const int i = mrow[w] / a.G, g = mrow[w] - i * a.G, hq = hk * a.G + g;
    R::frag(row[w].on ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qb + (int64_t)i * a.qs + (int64_t)hq * a.qh : nullptr, a.D, qf[w], lane);
    R::frag(row[w].on ? reinterpret_cast<const T*>(a.dout) + (int64_t)b * a.gb + (int64_t)i * a.gs + (int64_t)hq * a.gh : nullptr, a.D, gf[w], lane);
    lse[w] = row[w].on ? a.lse[(int64_t)bh * a.M + mrow[w]] : INFINITY;
    delta[w] = row[w].on ? a.delta[(int64_t)bh * a.M + mrow[w]] : 0.f;
  }
  const char* kbase = reinterpret_cast<const char*>(a.k) + ((int64_t)b * a.kb + (int64_t)hk * a.kh) * R::ES;
  const char* vbase = reinterpret_cast<const char*>(a.v) + ((int64_t)b * a.vb + (int64_t)hk * a.vh) * R::ES;
  const int64_t kst = a.ks * R::ES, vst = a.vs * R::ES;
  const int ltid = WK ? lane : tid;
  typename R::template Lin<C::LT> klin, vlin;
  klin.init(ltid, kst);
  vlin.init(ltid, vst);
  char* ring = smem + (WK ? wave * NS * C::SLOT : 0);
  auto issue = [&](int t, char* dst) {
    const bool holes = dw.holes;
    if (!holes && t * BN + BN <= a.Sk && a.D == DP) {
      klin.template load<BN>(dst, ltid, kbase + (int64_t)t * BN * kst, kst);
      vlin.template load<BN>(dst + C::TILE, ltid, vbase + (int64_t)t * BN * vst, vst);
      return;
    }
    R::template load2<BN, C::LT>(dst, dst + C::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
      const int key = t * BN + r;
      if (key >= a.Sk || (holes && a.kdoc[(int64_t)b * a.Sk + key] < 0)) return;
      p0 = kbase + (int64_t)key * a.ks * R::ES;
      p1 = vbase + (int64_t)key * a.vs * R::ES;
    });
  };
  f32x16 dq[RW][DT];
#pragma unroll
  for (int w = 0; w < RW; ++w)
#pragma unroll
    for (int j = 0; j < DT; ++j) dq[w][j] = zero16();

  struct Tile { int t; bool mixed; } q[NS];
  auto next = [&](int t) { return dw.template next<BN, STEP>(t, t1, 1, a.Sk, lane); };
  int slot = 0, fly = 0;
  auto fetch = [&](Tile& x, int t, int into) {
    x.t = next(t);
    x.mixed = dw.mixed;
    if (x.t < t1) { issue(x.t, ring + into * C::SLOT); ++fly; }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) fetch(q[i], i ? q[i - 1].t + STEP : (WK ? wave : 0), i);
  while (q[0].t < t1) {
    const int last = slot ? slot - 1 : NS - 1;
    if constexpr (WK) {
      fetch(q[NS - 1], q[NS - 2].t + STEP, last);
      vm_wait_tiles<C::NLD, NS - 1>(fly - 1);
    } else {
      vm_wait_tiles<C::NLD, NS - 2>(fly - 1);
      lds_barrier();
      fetch(q[NS - 1], q[NS - 2].t + STEP, last);
    }
    const char* kt = ring + slot * C::SLOT;
    const char* vt = kt + C::TILE;
    const bool mixed = q[0].mixed;
    const int k0 = q[0].t * BN;
    if (k0 < some) {
      f32x16 s[RW], dp[RW];
      R::template times<RW>(kt, 0, qf, s, lane);
      R::template times<RW>(vt, 0, gf, dp, lane);
      const bool caus = k0 + BN > whole;
      float mul = a.scale2;
      if (a.cap > 0.f) {
        tanh_all<T, RW>(s, a.icap);
        mul = a.cap2;
      }
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          dp[w][r] -= delta[w];
          if (a.cap > 0.f) dp[w][r] *= fmaf(-s[w][r], s[w][r], 1.f);
        }
      if (a.slopes) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
          const int at = row[w].pos - k0 - 4 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[w][r] = fmaf(-row[w].slope2, fabsf((float)(at - acc_row(r))), s[w][r] * mul);
        }
        mul = 1.f;
      }
      if (caus || mixed || k0 + BN > a.Sk) {
        const int key = k0 + (lane & 31), kd = mixed && key < a.Sk ? a.kdoc[(int64_t)b * a.Sk + key] : -1;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          int d = 0;
          if (mixed) d = __shfl(kd, acc_row(r) + 4 * h, 64);      // every lane gives its number
#pragma unroll
          for (int w = 0; w < RW; ++w) {
            const int last = min(caus ? max(row[w].pos, pre - 1) : a.Sk, a.Sk - 1) - k0 - 4 * h;
            const bool vis = acc_row(r) <= last && (!mixed || d == row[w].doc);
            s[w][r] = vis ? s[w][r] * mul : -INFINITY;
            dp[w][r] = vis ? dp[w][r] : 0.f;
          }
        }
        mul = 1.f;
      }
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[w][r] *= __builtin_amdgcn_exp2f(fmaf(s[w][r], mul, -lse[w]));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[RW][8];
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[w][e] = dp[w][8 * u + e];
        R::template t_times<RW, false>(kt, u * 16, x, dq, lane);
      }
    }
    if constexpr (WK) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    --fly;
    slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
    for (int i = 0; i + 1 < NS; ++i) q[i] = q[i + 1];
  }
  if constexpr (WK) join_waves<NW>(dq[0], reinterpret_cast<float*>(smem), wave, lane);
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    if (mrow[w] >= a.M) continue;
    const int i = mrow[w] / a.G, g = mrow[w] - i * a.G;
    const int64_t oi = (((int64_t)b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (WK && dt % NW != wave) continue;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d = dt * 32 + 8 * q4 + 4 * h;
        if (d >= a.D) continue;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = row[w].on ? dq[w][dt][4 * q4 + e] * a.scale : 0.f;
        R::put4(reinterpret_cast<T*>(a.dq) + oi + d, x);
      }
    }
  }
}

template <typename T, int DP, int NW, bool WK>
int run_dkv(Args& a, hipStream_t st) {
  typedef Dkv<T, DP, NW, WK> C;
  a.mtiles = (a.Sk + C::BK - 1) / C::BK;
  return launch(attn_dkv_kernel<T, DP, NW, WK>, (int64_t)a.mtiles * a.B * a.Hk, C::NT, C::LDS, a, st);
}
template <typename T, int DP, int NW, int RW, bool WK>
int run_dq(Args& a, hipStream_t st) {
  typedef Dq<T, DP, NW, RW, WK> C;
  a.mtiles = (a.M + C::BM - 1) / C::BM;
  return launch(attn_dq_kernel<T, DP, NW, RW, WK>, (int64_t)a.mtiles * a.B * a.Hk, C::NT, C::LDS, a, st);
}

template <typename T, int DP>
int bwd(Args& a, float* delta, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.Hq, bh = (int64_t)a.B * a.Hk;
  attn_delta_kernel<T><<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(a, delta);
  int rc = (int)hipGetLastError();
  if (rc) return rc;
  a.delta = delta;
  constexpr int WK = sizeof(T) == 4 && DP == 128 ? 2 : 4;
  if (a.dk) {
    const bool few = ((int64_t)a.Sk + 127) / 128 * bh < WKMAX;
    rc = few ? run_dkv<T, DP, WK, true>(a, st) : run_dkv<T, DP, 4, false>(a, st);
    if (rc) return rc;
  }
  if (!a.dq) return 0;
  const bool few = ((int64_t)a.M + 127) / 128 * bh < WKMAX;
  return few ? run_dq<T, DP, WK, 1, true>(a, st) : run_dq<T, DP, 4, 1, false>(a, st);
}

}  // namespace
}  // namespace turtle

using namespace turtle;

extern "C" int turtle_token_attn_bwd(const turtle_token_attn_grads* g, int dtype, void* stream) {
  Args a;
  if (!g || g->f.table || !fill(a, &g->f, dtype)) return -1;
  const int es = dtype == 0 ? 4 : 2;
  if (!rows16(g->dout, g->gb, g->gs, g->gh, es) || !a.lse || (!g->dk) != (!g->dv) || !g->delta) return -1;
  a.dout = g->dout; a.gb = g->gb; a.gs = g->gs; a.gh = g->gh;
  a.dq = g->dq; a.dk = g->dk; a.dv = g->dv;
  hipStream_t st = (hipStream_t)stream;
  const bool small = a.D <= 64;
  if (dtype == 0) return small ? bwd<float, 64>(a, g->delta, st) : bwd<float, 128>(a, g->delta, st);
  if (dtype == 1) return small ? bwd<bf16, 64>(a, g->delta, st) : bwd<bf16, 128>(a, g->delta, st);
  return small ? bwd<f16, 64>(a, g->delta, st) : bwd<f16, 128>(a, g->delta, st);
}
