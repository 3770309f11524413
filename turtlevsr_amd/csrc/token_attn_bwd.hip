// Token attention, backward (token_attn.h holds the method and the shared parts): delta, then dk and dv by key tiles,
// then dq by row tiles. No atomics: every sum has a fixed order.
#include "token_attn.h"
#ifndef KG128
#define KG128 0
#endif
#ifndef KWMIN
#define KWMIN (1<<30)
#endif
#ifndef QWMIN
#define QWMIN (1<<30)
#endif
#ifndef DKV_WAVES
#define DKV_WAVES (sizeof(T)==2 && KG==1 && DP==64 ? 2 : 1)
#endif
#ifndef DQ_WAVES
#define DQ_WAVES (sizeof(T)==2 && RW==1 ? 2 : 1)
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

template <typename T, int DP, int KG> struct Dkv {
  typedef Rows<T, DP> R;
  static constexpr int WKEYS = 32 * KG, BK = 4 * WKEYS;   // keys of a wave, of a block
  static constexpr int BM = 32;                           // rows of a tile
  static constexpr int TILE = BM * R::ROWB;
  static constexpr int STAGE = 2 * TILE + 64 * 4;         // Q, dO, 32 softmax sums and 32 deltas
  static constexpr int INFO = 3 * BM * 4;                 // place, document, slope of each row
  static constexpr int LDS = 2 * STAGE + 2 * INFO;
  static constexpr int NLD = R::template loads2<BM, 256>() + 1;
};

template <typename T, int DP, int KG>
__global__ __launch_bounds__(256, DKV_WAVES) void attn_dkv_kernel(Args a) {
  typedef Dkv<T, DP, KG> C;
  typedef Rows<T, DP> R;
  constexpr int BM = C::BM, DT = R::DT;
  // fp16: p times 2^10 as operand of dv (p of 10^4 keys would lose bits below the type's normal range)
  constexpr float POFF = std::is_same<T, f16>::value ? 10.f : 0.f, PS = std::is_same<T, f16>::value ? 1.f / 1024.f : 1.f;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int kt = item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int k0 = kt * C::BK, k1 = min(k0 + C::BK, a.Sk), off = a.Sk - a.Sq;
  const int kw = k0 + wave * C::WKEYS, kw1 = min(kw + C::WKEYS, a.Sk);
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
  constexpr int NI = BM * R::CH / 256;
  const bool plain = BM % a.G == 0 && a.D == DP;
  const int per = BM / a.G;
  int64_t qoff[NI], goff[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (i * 256 + tid) / R::CH, c = ((tid % R::CH) ^ R::swz(r)) << 4, ti = r / a.G, g = r - ti * a.G;
    qoff[i] = ((int64_t)ti * a.qs + (int64_t)g * a.qh) * R::ES + c;
    goff[i] = ((int64_t)ti * a.gs + (int64_t)g * a.gh) * R::ES + c;
  }
  auto issue = [&](int t, int stage) {
    char* dst = smem + stage * C::STAGE;
    if (rules && tid < 64) {
      const int m = t * BM + (lane & 31), i = m / a.G, g = m - i * a.G;
      float s = 0.f;
      if (a.slopes) s = a.G <= 64 ? __shfl(sl, g, 64) : a.slopes[hk * a.G + g] * LOG2E;
      int d = 0;
      if (dw.mixed) d = m < a.M ? a.qdoc[(int64_t)b * a.Sq + i] : -1;
      int* info = reinterpret_cast<int*>(smem + 2 * C::STAGE + stage * C::INFO);
      if (lane < BM) { info[lane] = i + off; info[BM + lane] = d; info[2 * BM + lane] = __float_as_int(s); }
    }
    const bool holes = dw.holes;
    if (plain && !holes && t * BM + BM <= a.M && (!a.causal || t * per + off >= 0 || pre > 0)) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t at = (uint32_t)(i * 256 + (tid & ~63)) * 16;
        dma16(qbase + qoff[i] + (int64_t)t * per * a.qs * R::ES, __builtin_amdgcn_readfirstlane(lds_addr(dst) + at));
        dma16(gbase + goff[i] + (int64_t)t * per * a.gs * R::ES, __builtin_amdgcn_readfirstlane(lds_addr(dst + C::TILE) + at));
      }
    } else
    R::template load2<BM, 256>(dst, dst + C::TILE, tid, a.D, [&](int r, const char*& p0, const char*& p1) {
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

  auto next = [&](int t) { return dw.template next<BM, 1>(t, t1, a.G, a.Sq, lane); };
  int t = next(t0), par = 0;
  if (t < t1) issue(t, 0);
  bool mixed = dw.mixed;
  while (t < t1) {
    const int tn = next(t + 1);
    if (tn < t1) {
      issue(tn, par ^ 1);
      vm_wait<C::NLD>();
    } else {
      vm_wait<0>();
    }
    lds_barrier();
    const char* qt = smem + par * C::STAGE;
    const char* gt = qt + C::TILE;
    const float* in = reinterpret_cast<const float*>(qt + 2 * C::TILE);
    const int* info = reinterpret_cast<const int*>(smem + 2 * C::STAGE + par * C::INFO);
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
    lds_barrier();
    par ^= 1;
    t = tn;
    mixed = dw.mixed;
  }
#pragma unroll
  for (int w = 0; w < KG; ++w) {
    if (key[w] >= a.Sk) continue;
    const int64_t oi = (((int64_t)b * a.Sk + key[w]) * a.Hk + hk) * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
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

template <typename T, int DP, int RW> struct Dq {
  typedef Rows<T, DP> R;
  static constexpr int WROWS = 32 * RW, BM = 4 * WROWS, BN = 32;
  static constexpr int TILE = BN * R::ROWB, LDS = 4 * TILE;
  static constexpr int NLD = R::template loads2<BN, 256>();
};

template <typename T, int DP, int RW>
__global__ __launch_bounds__(256, DQ_WAVES) void attn_dq_kernel(Args a) {
  typedef Dq<T, DP, RW> C;
  typedef Rows<T, DP> R;
  constexpr int BN = C::BN, DT = R::DT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int mt = a.mtiles - 1 - item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int off = a.Sk - a.Sq, m0 = mt * C::BM, m1 = min(m0 + C::BM, a.M);
  const int mw = m0 + wave * C::WROWS, mw1 = min(mw + C::WROWS, a.M);
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
  const int64_t koff = R::template lane_off<256>(tid, kst), voff = R::template lane_off<256>(tid, vst);
  auto issue = [&](int t, char* dst) {
    const bool holes = dw.holes;
    if constexpr (R::template linear<256>()) {
      if (!holes && t * BN + BN <= a.Sk && a.D == DP) {
        R::template load2_linear<BN, 256>(dst, dst + C::TILE, tid, kbase + koff + (int64_t)t * BN * kst, vbase + voff + (int64_t)t * BN * vst, kst, vst);
        return;
      }
    }
    R::template load2<BN, 256>(dst, dst + C::TILE, tid, a.D, [&](int r, const char*& p0, const char*& p1) {
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

  auto next = [&](int t) { return dw.template next<BN, 1>(t, t1, 1, a.Sk, lane); };
  int t = next(0), par = 0;
  if (t < t1) issue(t, smem);
  bool mixed = dw.mixed;
  while (t < t1) {
    const int tn = next(t + 1);
    if (tn < t1) {
      issue(tn, smem + (par ^ 1) * 2 * C::TILE);
      vm_wait<C::NLD>();
    } else {
      vm_wait<0>();
    }
    lds_barrier();
    const char* kt = smem + par * 2 * C::TILE;
    const char* vt = kt + C::TILE;
    const int k0 = t * BN;
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
    lds_barrier();
    par ^= 1;
    t = tn;
    mixed = dw.mixed;
  }
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    if (mrow[w] >= a.M) continue;
    const int i = mrow[w] / a.G, g = mrow[w] - i * a.G;
    const int64_t oi = (((int64_t)b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
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

template <typename T, int DP, int KG>
int run_dkv(Args& a, hipStream_t st) {
  typedef Dkv<T, DP, KG> C;
  a.mtiles = (a.Sk + C::BK - 1) / C::BK;
  return launch(attn_dkv_kernel<T, DP, KG>, (int64_t)a.mtiles * a.B * a.Hk, 256, C::LDS, a, st);
}
template <typename T, int DP, int RW>
int run_dq(Args& a, hipStream_t st) {
  typedef Dq<T, DP, RW> C;
  a.mtiles = (a.M + C::BM - 1) / C::BM;
  return launch(attn_dq_kernel<T, DP, RW>, (int64_t)a.mtiles * a.B * a.Hk, 256, C::LDS, a, st);
}

template <typename T, int DP>
int bwd(Args& a, float* delta, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.Hq, bh = (int64_t)a.B * a.Hk;
  attn_delta_kernel<T><<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(a, delta);
  int rc = (int)hipGetLastError();
  if (rc) return rc;
  a.delta = delta;
  constexpr int W2 = sizeof(T) == 2 && (DP == 64 || KG128) ? 2 : 1;
  const bool kw = W2 == 2 && (a.Sk + 255) / 256 * bh >= KWMIN, qw = W2 == 2 && (a.M + 255) / 256 * bh >= QWMIN;
  if (a.dk) {
    rc = kw ? run_dkv<T, DP, W2>(a, st) : run_dkv<T, DP, 1>(a, st);
    if (rc) return rc;
  }
  if (!a.dq) return 0;
  return qw ? run_dq<T, DP, W2>(a, st) : run_dq<T, DP, 1>(a, st);
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
