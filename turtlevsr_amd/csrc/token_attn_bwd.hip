// Token attention, backward (token_attn.h holds the method and the shared parts): delta, then dk and dv by key tiles,
// then dq by row tiles, then the sums of split walks. No atomics: every sum has a fixed order.
//
// Two kernels compute S and dP twice (14 products of a tile pair for 10) and in exchange neither dk, dv nor dq is ever
// summed through memory. A wave's step is a chain - S and dP, the rules, the exponential, two products with the results -
// so with two waves on a SIMD what counts is the chain's waits: LDS reads started ahead of their products (dq at 128
// channels 400 -> 365 us, dk and dv at 64 channels 212 -> 188), masks without branches (packed documents 850 -> 690).
// Measured, bf16: 2 x 5120 tokens causal with prefix 2048, 8 heads of 64 channels: dk, dv 182 us (4 products a pair, 686
// TF/s), dq 125 us (3 products, 750 TF/s), delta 9 us; 7 documents in 8192 tokens, 16 heads on 4 of 128 channels: dk, dv
// 495 us and 25 for their sums, dq 359 us, delta 17 us (whole walks instead of split ones take 20 % more: the block over the
// border of the longest documents walks 2.5 times the mean block's way). fp32, 2 x 333 on 517 tokens, 6 heads on 3 of 48
// channels: 33, 22, 5 us.
#include "token_attn.h"

namespace turtle {
namespace {

__device__ const float g_row_pad[2] = {INFINITY, 0.f};   // softmax sum and delta of a row that is not there

// -delta [B][Hk][M], delta = do . (o + o_lo); 8 lanes a row, 16 bytes a lane and step. A row that sees nothing may hold
// anything, in q and in do: its delta is 0, and with documents its tile is marked as one with holes, so that dk's and dv's
// kernel asks for each row (every backward writes the same mark).
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(Args a, float* delta) {
  constexpr int V = 16 / sizeof(T);
  const int64_t u = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int64_t n = (int64_t)a.B * a.Sq * a.Hq;
  const int ln = threadIdx.x & 7;
  float s = 0.f;
  if (u < n) {
    const int64_t b = u / ((int64_t)a.Sq * a.Hq), j = u - b * a.Sq * a.Hq, i = j / a.Hq, hq = j - i * a.Hq;
    const int64_t at = ((b * a.Hk + hq / a.G) * a.Sq + i) * a.G + hq % a.G;
    const T* g = reinterpret_cast<const T*>(a.dout) + b * a.gb + i * a.gs + hq * a.gh;
    const T* o = reinterpret_cast<const T*>(a.o) + u * a.D;
    const T* lo = a.olo ? reinterpret_cast<const T*>(a.olo) + u * a.D : nullptr;
    const bool blind = a.lse[at] == INFINITY;
    typedef T tv __attribute__((ext_vector_type(V)));
    for (int d = ln * V; d < a.D; d += 8 * V) {
      const tv x = *reinterpret_cast<const tv*>(g + d), y = *reinterpret_cast<const tv*>(o + d);
      tv z = {};
      if (lo) z = *reinterpret_cast<const tv*>(lo + d);
#pragma unroll
      for (int e = 0; e < V; ++e) s = fmaf((float)x[e], (float)y[e] + (float)z[e], s);
    }
    s += __shfl_xor(s, 1, 64); s += __shfl_xor(s, 2, 64); s += __shfl_xor(s, 4, 64);
    if (ln == 0) {
      delta[at] = blind ? 0.f : -s;
      if (blind && a.qdoc) const_cast<int4*>(a.qr)[b * a.nqr + i / RT].w = 1;
    }
  }
}

// WK: for small grids - the block's NW waves own the same 32 keys and take the row tiles in turn, each with its own
// ring and no barriers, and join at the end.
// 128 channels: the operands of S and dP and the two accumulators take 192 registers of the 256 that two waves of a
// SIMD can have, and one wave alone leaves its latencies bare. RG = 2: two waves share 32 keys, take half of every row
// tile each and join at the end; V stays in LDS. SP (fp32, and the small grids): a block computes dk (S, dP, dk) or dv
// (S, dv), 40 products for 32.
template <typename T, int DP, int NW, int RG, bool WK> struct Dkv {
  typedef Rows<T, DP> R;
  static constexpr int NT = NW * RG * 64, LT = WK ? 64 : NT;
  static constexpr int BK = WK ? 32 : NW * 32;            // keys of a block
  static constexpr bool SP = DP == 128 && RG == 1, VL = RG > 1;
  static constexpr int MT = (sizeof(T) == 2 && DP == 64 && !WK) ? 2 : 1, WM = 32 * MT;    // rows a wave takes of a tile
  static constexpr int BM = WM * RG;                      // rows of a tile
  static constexpr int NS = (WK || DP == 128) ? 2 : 3;
  static constexpr int TILE = BM * R::ROWB;
  static constexpr int SLOT = (2 * TILE + 4 * BM * 4 + 256 + 511) / 512 * 512;      // Q, dO; softmax sum, delta, place, slope, document of a row
  static constexpr int RING = NS * SLOT * (WK ? NW : 1), JOIN = R::DT * 16 * 64 * 4 * (RG > 1 ? NW : 1);
  static constexpr int LDS = (RING > JOIN ? RING : JOIN) + (VL ? BK * R::ROWB : 0);
  static constexpr int NLD = R::template loads2<BM, LT>() + BM / 32;
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

// dS as an fp16 operand of dk (dq) is taken times 2^e: unscaled, a pair among 4096 keys under a dO of 1e-3 is near the type's
// smallest numbers (dq off by 0.5 %, by 5 % at 1e-4), and one of a large dO past 65504. e belongs to the key (row) that a
// lane and lane ^ 32 own, one column of the accumulators. It starts at 60, falls when a |dS| 2^e passes 2^15 - to where the
// largest one is under 2^8 - and never rises, so what is lost lies 2^-32 below the column's largest dS. Powers of two:
// the sums are scaled over without an error, and no lane's result depends on another column's.
template <typename T> struct Lift {
  static constexpr bool on = std::is_same<T, f16>::value;
  int e;
  TURTLE_DEV static float pow2(int n) { return __int_as_float((127 + n) << 23); }
  // ds of a tile, times 2^e; acc: the sums of the tiles before
  template <int N, int DT>
  TURTLE_DEV void fit(f32x16 (&ds)[N], f32x16 (&acc)[DT]) {
    if constexpr (!on) return;
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(ds[j][r]));
    if (__any(big * pow2(e) > 32768.f)) {
      big = half_max(big);
      const int to = big * pow2(e) > 32768.f ? min(e, 8 - __builtin_amdgcn_frexp_expf(big)) : e;      // -120 at least
      const float f = ldexpf(1.f, to - e);
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
      e = to;
    }
    const float up = pow2(e);
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[j][r] *= up;
  }
  // the sums as they are
  template <int DT>
  TURTLE_DEV void drop(f32x16 (&acc)[DT]) const {
    if constexpr (!on) return;
    const float down = pow2(-e);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= down;
  }
};

// dv's accumulators: its own, or dk's where a block has only one of them
template <bool SAME, int N, int M>
TURTLE_DEV auto& pick(f32x16 (&x)[N], f32x16 (&y)[M]) {
  if constexpr (SAME) return x;
  else return y;
}

template <typename T, int DP, int NW, int RG, bool WK, bool SPLIT>
__global__ __launch_bounds__(NW * RG * 64, sizeof(T) == 2 && (DP == 64 || RG == 2) ? 2 : 1) void attn_dkv_kernel(Args a) {
  typedef Dkv<T, DP, NW, RG, WK> C;
  typedef Rows<T, DP> R;
  constexpr int BM = C::BM, MT = C::MT, DT = R::DT, NS = C::NS, STEP = WK ? NW : 1;
  // fp16: p times 2^10 as operand of dv (p of 10^4 keys would lose bits below the type's normal range)
  constexpr float PUP = std::is_same<T, f16>::value ? 1024.f : 1.f;
  extern __shared__ __attribute__((aligned(512))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wv % NW, rg = wv / NW, h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  constexpr bool SP = C::SP;
  const bool do_k = !SP || !(item & 1), do_v = !SP || (item & 1);
  const int nsplit = SPLIT ? a.nsplit : 1, ik = SP ? item >> 1 : item, is = ik / nsplit, sp = ik - is * nsplit, step = STEP * nsplit;
  const int kt = is % a.mtiles, bh = is / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int k0 = kt * C::BK, k1 = min(k0 + C::BK, a.Sk), off = a.Sk - a.Sq;
  const int kw = k0 + (WK ? 0 : wave * 32), kw1 = min(kw + 32, a.Sk);
  const int pre = a.prefix ? max(a.prefix[b], 0) : 0;
  const int key = kw + (lane & 31);
  int kdoc = (a.kdoc && key < a.Sk) ? a.kdoc[(int64_t)b * a.Sk + key] : 0;
  const bool kon = key < a.Sk && kdoc >= 0;
  uint4 kf[R::STEPS], vf[R::STEPS];
  R::frag(kon ? reinterpret_cast<const T*>(a.k) + (int64_t)b * a.kb + (int64_t)key * a.ks + (int64_t)hk * a.kh : nullptr, a.D, kf, lane);
  R::frag(kon ? reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vb + (int64_t)key * a.vs + (int64_t)hk * a.vh : nullptr, a.D, vf, lane);
  arrived(kdoc);
  char* vlds = smem + C::LDS - C::BK * R::ROWB + wave * 32 * R::ROWB;
  if constexpr (C::VL) {
    // V's chunks at the places `chunk` reads them from; every row group writes the same
#pragma unroll
    for (int s = 0; s < R::STEPS; ++s)
      *reinterpret_cast<uint4*>(vlds + (lane & 31) * R::ROWB + (((2 * s + h) ^ R::swz(lane & 31)) << 4)) = vf[s];
  }

  // rows that may see a key of this block
  int mfirst = 0;
  if (a.causal && k0 >= pre) mfirst = max(0, k0 - off) * a.G;
  const int t1 = (a.M + BM - 1) / BM, t0 = min(t1, mfirst / BM);
  DocWalk dw;
  dw.none();
  if (a.qdoc) dw.init(a.qr + (int64_t)b * a.nqr, a.nqr, doc_range(a.kr + (int64_t)b * a.nkr, a.nkr, k0, k1));
  float sl = (a.slopes && lane < a.G) ? a.slopes[hk * a.G + lane] * LOG2E : 0.f;
  arrived(sl);
  const bool rules = a.causal || a.slopes || a.qdoc;

  const char* qbase = reinterpret_cast<const char*>(a.q) + ((int64_t)b * a.qb + (int64_t)hk * a.G * a.qh) * R::ES;
  const char* gbase = reinterpret_cast<const char*>(a.dout) + ((int64_t)b * a.gb + (int64_t)hk * a.G * a.gh) * R::ES;
  // where a tile holds whole tokens, its rows lie at the same offsets from its first one every time
  const int ltid = WK ? lane : tid;
  constexpr int NI = BM * R::CH / C::LT;
  const bool plain = BM % a.G == 0 && a.D == DP;
  const int per = token_of(a, BM);
  int64_t qoff[NI], goff[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (i * C::LT + ltid) / R::CH, c = ((ltid % R::CH) ^ R::swz(r)) << 4, ti = token_of(a, r), g = r - ti * a.G;
    qoff[i] = ((int64_t)ti * a.qs + (int64_t)g * a.qh) * R::ES + c;
    goff[i] = ((int64_t)ti * a.gs + (int64_t)g * a.gh) * R::ES + c;
  }
  const int64_t qstep = (int64_t)per * a.qs * R::ES, gstep = (int64_t)per * a.gs * R::ES;
  const float* sums = a.lse + (int64_t)bh * a.M;
  const float* deltas = a.delta + (int64_t)bh * a.M;
  char* ring = smem + (WK ? wave * NS * C::SLOT : 0);
  auto issue = [&](int t, char* dst) __attribute__((always_inline)) {
    if (dw.mixed) {
      const int m = t * BM + (lane & (BM - 1));
      dma4(m < a.M ? a.qdoc + (int64_t)b * a.Sq + token_of(a, m) : &g_no_doc, __builtin_amdgcn_readfirstlane(lds_addr(dst + 2 * C::TILE + 16 * BM)));
    }
    const int m = t * BM + ltid, i = token_of(a, m), g = m - i * a.G;
    float s = 0.f;
    if (a.slopes) s = a.G <= 64 ? __shfl(sl, g & 63, 64) : a.slopes[hk * a.G + g] * LOG2E;      // by all lanes: each gives one
    if (rules && ltid < BM) {
      int* info = reinterpret_cast<int*>(dst + 2 * C::TILE) + 2 * BM + ltid;
      info[0] = i + off;
      info[BM] = __float_as_int(s);
    }
    const int m0 = t * BM;
    if (plain && !dw.holes && m0 + BM <= a.M && (!a.causal || t * per + off >= 0 || pre > 0)) {
      const char *qp = qbase + t * qstep, *gp = gbase + t * gstep;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t at = (uint32_t)(i * C::LT + (ltid & ~63)) * 16;
        dma16(qp + qoff[i], __builtin_amdgcn_readfirstlane(lds_addr(dst) + at));
        dma16(gp + goff[i], __builtin_amdgcn_readfirstlane(lds_addr(dst + C::TILE) + at));
      }
    } else {
      const bool holes = dw.holes;
      R::template load2<BM, C::LT>(dst, dst + C::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
        const int m = m0 + r, i = token_of(a, m), g = m - i * a.G;
        // rows that see nothing may hold anything: they are not read
        if (m >= a.M || (a.causal && i + off < 0 && pre <= 0) || (holes && sums[m] == INFINITY)) return;
        p0 = qbase + ((int64_t)i * a.qs + (int64_t)g * a.qh) * R::ES;
        p1 = gbase + ((int64_t)i * a.gs + (int64_t)g * a.gh) * R::ES;
      });
    }
    // every wave writes the same sums and deltas, so that all count the same number of loads
#pragma unroll
    for (int j = 0; j < BM / 32; ++j) {
      const int e = j * 64 + lane, mr = m0 + (e & (BM - 1)), which = e / BM;
      const float* src = mr < a.M ? (which ? deltas : sums) + mr : g_row_pad + which;
      dma4(src, __builtin_amdgcn_readfirstlane(lds_addr(dst + 2 * C::TILE) + j * 256));
    }
  };

  // the sums of dk and dv; SP: the one or the other
  f32x16 dk[DT], dv_[SP ? 1 : DT];
  auto& dv = pick<SP>(dk, dv_);
#pragma unroll
  for (int i = 0; i < DT; ++i) { dk[i] = zero16(); dv[i] = zero16(); }
  Lift<T> lift{60};

  // the walk over row tiles: as the forward's over key tiles
  struct Tile { int t; bool mixed; } q[NS - 1];
  int tnew = t0 + sp * STEP + (WK ? wave : 0), fly = 0, into = 0, slot = 0;
  auto start = [&]() __attribute__((always_inline)) {
    Tile x{dw.template next<BM>(tnew, t1, step, a.G, a.Sq, lane), false};
    x.mixed = dw.mixed;
    if (x.t < t1) { issue(x.t, ring + into * C::SLOT); ++fly; }
    tnew = x.t + step;
    into = into + 1 == NS ? 0 : into + 1;
#pragma unroll
    for (int i = 0; i + 2 < NS; ++i) q[i] = q[i + 1];
    q[NS - 2] = x;
  };
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) start();
  arrived(kf);
  if constexpr (!C::VL) arrived(vf);
  for (;;) {
    const Tile cur = q[0];
    if (cur.t >= t1) break;
    if constexpr (!WK) {
      vm_wait_tiles<C::NLD, NS - 2>(fly - 1);
      lds_barrier();
    }
    start();
    if constexpr (WK) vm_wait_tiles<C::NLD, NS - 1>(fly - 1);
    const char* qt = ring + slot * C::SLOT + rg * C::WM * R::ROWB;      // this wave's rows of the tile
    const char* gt = qt + C::TILE;
    const float* in = reinterpret_cast<const float*>(ring + slot * C::SLOT + 2 * C::TILE) + rg * C::WM + 4 * h;
    const int* info = reinterpret_cast<const int*>(in) + 2 * BM;
    const bool mixed = cur.mixed;
    // causal: places of the first and last row
    const int m0 = cur.t * BM + rg * C::WM, m1 = min(m0 + C::WM, a.M);
    const int p0 = token_of(a, m0) + off, p1 = token_of(a, max(m1 - 1, 0)) + off;
    if (m0 < m1 && (!a.causal || p1 >= kw || kw < pre) && kw < a.Sk) {
      // dP starts from -delta (stored negated)
      f32x16 s[MT], dp[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 del = *reinterpret_cast<const float4*>(in + BM + j * 32 + 8 * c);
          dp[j][4 * c] = del.x; dp[j][4 * c + 1] = del.y; dp[j][4 * c + 2] = del.z; dp[j][4 * c + 3] = del.w;
        }
      if constexpr (C::VL) R::times2_lds(qt, gt, kf, vlds, s[0], dp[0], lane);
      else if (do_k) R::template times2<MT>(qt, gt, kf, vf, s, dp, lane);
      else R::template times<MT>(qt, kf, s, lane);
      const bool caus = a.causal && p0 + 1 < kw1 && kw1 > pre;
      float mul = a.scale2;
      if (a.cap > 0.f) {
        tanh_all<T, MT>(s, a.icap, a.cap);
        mul = a.cap2;
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[j][r] *= fmaf(-s[j][r], s[j][r], 1.f);      // times the cap's slope
      }
      if (a.slopes) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int4 pos = *reinterpret_cast<const int4*>(info + j * 32 + 8 * c);
            const float4 slp = *reinterpret_cast<const float4*>(info + BM + j * 32 + 8 * c);
            const int po[4] = {pos.x, pos.y, pos.z, pos.w};
            const float sp[4] = {slp.x, slp.y, slp.z, slp.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][4 * c + e] = fmaf(-sp[e], fabsf((float)(po[e] - key)), s[j][4 * c + e] * mul);
          }
        mul = 1.f;
      }
      // the pairs that do not see each other: p = 0, whatever dP holds there (a pass for each rule, free of branches)
      if (caus || mixed) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] *= mul;
        mul = 1.f;
      }
      auto hide = [&](const int* at, auto sees) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int4 x = *reinterpret_cast<const int4*>(at + j * 32 + 8 * c);
            const int y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool vis = sees(y[e]);
              s[j][4 * c + e] = vis ? s[j][4 * c + e] : -INFINITY;
              dp[j][4 * c + e] = vis ? dp[j][4 * c + e] : 0.f;
            }
          }
      };
      if (caus) {
        const int from = key < pre ? -0x7fffffff - 1 : key;      // the first place that sees the key
        hide(info, [&](int place) { return place >= from; });
      }
      if (mixed) hide(info + 2 * BM, [&](int doc) { return doc == kdoc; });
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 lse = *reinterpret_cast<const float4*>(in + j * 32 + 8 * c);
          const float ls[4] = {lse.x, lse.y, lse.z, lse.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * c + e;
            s[j][r] = __builtin_amdgcn_exp2f(fmaf(s[j][r], mul, -ls[e]));
            dp[j][r] *= s[j][r];
            if constexpr (PUP != 1.f) s[j][r] *= PUP;
          }
        }
      if (do_v) R::template t_times_all<MT>(gt, s, dv, lane);
      if (do_k) {
        lift.fit(dp, dk);
        R::template t_times_all<MT>(qt, dp, dk, lane);
      }
    }
    if constexpr (WK) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    --fly;
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  if (do_k) lift.drop(dk);
  if constexpr (WK) {
    join_waves<NW>(dk, reinterpret_cast<float*>(smem), wave, lane);
    if constexpr (!SP) join_waves<NW>(dv, reinterpret_cast<float*>(smem), wave, lane);
  }
  if constexpr (RG > 1) {
    // the row groups' sums, in order, through LDS
    float* sum = reinterpret_cast<float*>(smem) + wave * DT * 16 * 64 + lane;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f32x16 (&acc)[DT] = k ? dv : dk;
      __syncthreads();
      if (rg == 1) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[(dt * 16 + r) * 64] = acc[dt][r];
      }
      __syncthreads();
      if (rg == 0) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[dt][r] += sum[(dt * 16 + r) * 64];
      }
    }
    if (rg > 0) return;
  }
  if (key >= a.Sk) return;
  const int64_t oi = (((int64_t)b * a.Sk + key) * a.Hk + hk) * a.D;
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
        x[e] = kon ? dk[dt][4 * q4 + e] * a.scale : 0.f;
        y[e] = kon ? dv[dt][4 * q4 + e] * (1.f / PUP) : 0.f;
      }
      if constexpr (SPLIT) {
        float* part = a.part + (int64_t)sp * 2 * a.B * a.Sk * a.Hk * a.D + oi + d;
        if (do_k) *reinterpret_cast<float4*>(part) = make_float4(x[0], x[1], x[2], x[3]);
        if (do_v) *reinterpret_cast<float4*>(part + (int64_t)a.B * a.Sk * a.Hk * a.D) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        if (do_k) R::put4(reinterpret_cast<T*>(a.dk) + oi + d, x);
        if (do_v) R::put4(reinterpret_cast<T*>(a.dv) + oi + d, y);
      }
    }
  }
}

template <typename T, int DP, int NW, bool WK> struct Dq {
  typedef Rows<T, DP> R;
  static constexpr int NT = NW * 64, LT = WK ? 64 : NT;
  static constexpr int BM = WK ? 32 : NW * 32;            // rows of a block
  static constexpr int KT = (sizeof(T) == 2 && DP == 64) ? 2 : 1, BN = 32 * KT;      // keys of a tile
  static constexpr int NS = WK ? 2 : 3;
  static constexpr int TILE = BN * R::ROWB, SLOT = 2 * TILE + 512;      // K, V; document of a key
  static constexpr int RING = NS * SLOT * (WK ? NW : 1), JOIN = R::DT * 16 * 64 * 4;
  static constexpr int LDS = RING > JOIN ? RING : JOIN;
  static constexpr int NLD = R::template loads2<BN, LT>();
};

template <typename T, int DP, int NW, bool WK, bool SPLIT>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(Args a) {
  typedef Dq<T, DP, NW, WK> C;
  typedef Rows<T, DP> R;
  constexpr int BN = C::BN, KT = C::KT, DT = R::DT, NS = C::NS, STEP = WK ? NW : 1;
  extern __shared__ __attribute__((aligned(512))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int nsplit = SPLIT ? a.nsplit : 1, is = item / nsplit, sp = item - is * nsplit, step = STEP * nsplit;
  const int mt = a.mtiles - 1 - is % a.mtiles, bh = is / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int off = a.Sk - a.Sq, m0 = mt * C::BM, m1 = min(m0 + C::BM, a.M);
  const int mw = m0 + (WK ? 0 : wave * 32), mw1 = min(mw + 32, a.M);
  const int pre = a.prefix ? max(a.prefix[b], 0) : 0;
  int kend = a.Sk;
  if (a.causal) kend = min(a.Sk, max(token_of(a, m1 - 1) + off + 1, pre));
  const int t1 = (max(kend, 0) + BN - 1) / BN;
  // what this wave's rows see whole: keys before `whole`; and at all: keys before `some`
  const int whole = a.causal ? max(token_of(a, mw) + off + 1, pre) : 0x7fffffff;
  const int some = mw1 <= mw ? 0 : (a.causal ? max(token_of(a, mw1 - 1) + off + 1, pre) : 0x7fffffff);

  const int mrow = mw + (lane & 31);
  Row row = row_of(a, b, hk, mrow, off, a.Sq);
  DocWalk dw;
  dw.none();
  if (a.qdoc)
    dw.init(a.kr + (int64_t)b * a.nkr, a.nkr, doc_range(a.qr + (int64_t)b * a.nqr, a.nqr, token_of(a, m0), token_of(a, m1 - 1) + 1));
  const int i = token_of(a, mrow), g = mrow - i * a.G, hq = hk * a.G + g;
  uint4 qf[R::STEPS], gf[R::STEPS];
  R::frag(row.on ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qb + (int64_t)i * a.qs + (int64_t)hq * a.qh : nullptr, a.D, qf, lane);
  R::frag(row.on ? reinterpret_cast<const T*>(a.dout) + (int64_t)b * a.gb + (int64_t)i * a.gs + (int64_t)hq * a.gh : nullptr, a.D, gf, lane);
  float lse = row.on ? a.lse[(int64_t)bh * a.M + mrow] : INFINITY, delta = row.on ? a.delta[(int64_t)bh * a.M + mrow] : 0.f;

  const char* kbase = reinterpret_cast<const char*>(a.k) + ((int64_t)b * a.kb + (int64_t)hk * a.kh) * R::ES;
  const char* vbase = reinterpret_cast<const char*>(a.v) + ((int64_t)b * a.vb + (int64_t)hk * a.vh) * R::ES;
  const int64_t kst = a.ks * R::ES, vst = a.vs * R::ES;
  const int ltid = WK ? lane : tid;
  typename R::template Lin<C::LT> klin, vlin;
  klin.init(ltid, kst);
  vlin.init(ltid, vst);
  char* ring = smem + (WK ? wave * NS * C::SLOT : 0);
  auto issue = [&](int t, char* dst) __attribute__((always_inline)) {
    const int k0 = t * BN;
    if (dw.mixed) key_docs<BN>(a, b, k0, dst + 2 * C::TILE, lane);
    if (!dw.holes && k0 + BN <= a.Sk && a.D == DP) {
      klin.template load<BN>(dst, ltid, kbase + k0 * kst, kst);
      vlin.template load<BN>(dst + C::TILE, ltid, vbase + k0 * vst, vst);
      return;
    }
    const bool holes = dw.holes;
    R::template load2<BN, C::LT>(dst, dst + C::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
      const int key = k0 + r;
      if (key >= a.Sk || (holes && a.kdoc[(int64_t)b * a.Sk + key] < 0)) return;
      p0 = kbase + key * kst;
      p1 = vbase + key * vst;
    });
  };
  f32x16 dq[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j) dq[j] = zero16();
  Lift<T> lift{60};

  struct Tile { int t; bool mixed; } q[NS - 1];
  int tnew = sp * STEP + (WK ? wave : 0), fly = 0, into = 0, slot = 0;
  auto start = [&]() __attribute__((always_inline)) {
    Tile x{dw.template next<BN>(tnew, t1, step, 1, a.Sk, lane), false};
    x.mixed = dw.mixed;
    if (x.t < t1) { issue(x.t, ring + into * C::SLOT); ++fly; }
    tnew = x.t + step;
    into = into + 1 == NS ? 0 : into + 1;
#pragma unroll
    for (int j = 0; j + 2 < NS; ++j) q[j] = q[j + 1];
    q[NS - 2] = x;
  };
#pragma unroll 1
  for (int j = 0; j < NS - 1; ++j) start();
  arrived(qf);
  arrived(gf);
  arrived(lse);
  arrived(delta);
  arrived(row.doc);
  arrived(row.slope2);
  f32x16 ndelta;      // dP starts from -delta (stored negated)
#pragma unroll
  for (int r = 0; r < 16; ++r) ndelta[r] = delta;
  for (;;) {
    const Tile cur = q[0];
    if (cur.t >= t1) break;
    if constexpr (!WK) {
      vm_wait_tiles<C::NLD, NS - 2>(fly - 1);
      lds_barrier();
    }
    start();
    if constexpr (WK) vm_wait_tiles<C::NLD, NS - 1>(fly - 1);
    const char* kt = ring + slot * C::SLOT;
    const char* vt = kt + C::TILE;
    const int k0 = cur.t * BN;
    const bool mixed = cur.mixed;
    if (k0 < some) {
      f32x16 s[KT], dp[KT];
#pragma unroll
      for (int j = 0; j < KT; ++j) dp[j] = ndelta;
      R::template times2<KT>(kt, vt, qf, gf, s, dp, lane);
      float mul = a.scale2;
      if (a.cap > 0.f) {
        tanh_all<T, KT>(s, a.icap, a.cap);
        mul = a.cap2;
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[j][r] *= fmaf(-s[j][r], s[j][r], 1.f);      // times the cap's slope
      }
      if (a.slopes) {
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int at = row.pos - k0 - j * 32 - 4 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = fmaf(-row.slope2, fabsf((float)(at - acc_row(r))), s[j][r] * mul);
        }
        mul = 1.f;
      }
      if (k0 + BN > whole || mixed || k0 + BN > a.Sk) {
        // the last key in sight; the pairs that do not see each other: p = 0, whatever dP holds there
        const int last = min(a.causal ? max(row.pos, pre - 1) : a.Sk, a.Sk - 1) - k0 - 4 * h;
        const int* kd = reinterpret_cast<const int*>(kt + 2 * C::TILE) + 4 * h;
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            int4 doc = make_int4(row.doc, row.doc, row.doc, row.doc);
            if (mixed) doc = *reinterpret_cast<const int4*>(kd + j * 32 + 8 * c);
            const int dc[4] = {doc.x, doc.y, doc.z, doc.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * c + e;
              const bool vis = j * 32 + acc_row(r) <= last && dc[e] == row.doc;
              s[j][r] = vis ? s[j][r] * mul : -INFINITY;
              dp[j][r] = vis ? dp[j][r] : 0.f;
            }
          }
        mul = 1.f;
      }
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[j][r] *= __builtin_amdgcn_exp2f(fmaf(s[j][r], mul, -lse));
      lift.fit(dp, dq);
      R::template t_times_all<KT>(kt, dp, dq, lane);
    }
    if constexpr (WK) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    --fly;
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  lift.drop(dq);
  if constexpr (WK) join_waves<NW>(dq, reinterpret_cast<float*>(smem), wave, lane);
  if (mrow >= a.M) return;
  const int64_t oi = (((int64_t)b * a.Sq + i) * a.Hq + hq) * a.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if (WK && dt % NW != wave) continue;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * h;
      if (d >= a.D) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = row.on ? dq[dt][4 * q4 + e] * a.scale : 0.f;
      if constexpr (SPLIT) *reinterpret_cast<float4*>(a.part + (int64_t)sp * a.B * a.Sq * a.Hq * a.D + oi + d) = make_float4(x[0], x[1], x[2], x[3]);
      else R::put4(reinterpret_cast<T*>(a.dq) + oi + d, x);
    }
  }
}

// the splits' sums of one kernel -> o0 (first half of a split's values) and, if there, o1, of n values each
struct Sum {
  const float* part;
  void *o0, *o1;
  int64_t n;
  int nsplit;
};

// both kernels' (blockIdx.y), 4 values a thread
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(Sum kv, Sum q) {
  const Sum a = blockIdx.y ? q : kv;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, all = a.o1 ? 2 * a.n : a.n;
  if (i >= all) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(a.part + s * all + i);
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
  }
  Rows<T, 64>::put4(i < a.n ? reinterpret_cast<T*>(a.o0) + i : reinterpret_cast<T*>(a.o1) + (i - a.n), v);
}

// The shape of a backward kernel. few: a block's waves own 32 keys (rows) together (WK) instead of 32 each: four times the
// blocks. Measured at 1024 tokens and 8, 16, 24 and 32 heads (64 .. 256 blocks of 128), us with / without:
//   dk, dv  bf16, 64 channels 21 / 40, 24 / 40, 39 / 42, 43 / 43; 128 channels 46 / 48, 91 / 51, 132 / 53, 176 / 56
//           fp32, 64 channels 58 / 181, 112 / 184, 165 / 187, 222 / 190; 128 channels 268 / 258 (32 blocks 135 / 255), 536 / 265
//   dq      bf16, 64 channels 11 / 22, 20 / 22, 28 / 23, 37 / 24; 128 channels 18 / 40, 36 / 41, 52 / 42, 69 / 44
//           fp32, 64 channels 40 / 128, 77 / 131, 115 / 135, 156 / 137; 128 channels 129 / 242, 261 / 247
// split: blocks take every split-th tile of the walk, 2 at least for each wave, and a second kernel adds up their fp32
// sums: where the blocks are fewer than the CUs (bf16 of 128 channels, 3 rows on 9000 keys, 2 heads, dq 84 us without, 14 + 4
// with; 8192 rows on 64 keys, dk and dv 120, 19 + 5; 1024 tokens, 1 head, dk and dv 24, 15 + 4), and with documents, where
// walks differ in length, up to four times as many (8192 tokens in 7 documents of 29 to 2535, 16 heads on 4, dk and
// dv 674 us without, 576 + 13 split in two, 504 + 23 in four; in 4 of 2048, 403, 405 + 13, 417 + 22). Full grids
// without documents gain nothing (1024 tokens, 8 heads to twice the CUs: dq 18 us, 28 + 4).
struct Shape { bool few; int split; };
Shape shape_of(const In* x, int dtype, bool dq) {
  const bool half = dtype != 0, wide = x->D > 64;
  const int64_t M = (int64_t)x->Sq * (x->Hq / x->Hk), own = dq ? M : x->Sk, walk = dq ? x->Sk : M, bh = (int64_t)x->B * x->Hk;
  Shape p;
  p.few = (own + 127) / 128 * bh <= (dq && half ? 128 : wide ? 64 : 255);
  const int64_t blocks = (own + (p.few ? 31 : 127)) / (p.few ? 32 : 128) * bh * (!dq && wide && (p.few || !half) ? 2 : 1);
  const int64_t tiles = (walk + 31) / 32 / (p.few ? (half || !wide ? 4 : 2) : 1);      // of a wave, about
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>({(x->qdoc ? 1024 : 256) / blocks, tiles / 2, 16}));
  return p;
}

// bytes of a kernel's sums, 0 where it is not split
size_t part_bytes(const In* x, int dtype, bool dq) {
  const int split = shape_of(x, dtype, dq).split;
  return split > 1 ? (size_t)split * x->B * (dq ? (size_t)x->Sq * x->Hq : (size_t)2 * x->Sk * x->Hk) * x->D * sizeof(float) : 0;
}

template <typename T, int DP, int NW, int RG, bool WK>
int run_dkv(Args& a, hipStream_t st) {
  typedef Dkv<T, DP, NW, RG, WK> C;
  a.mtiles = (a.Sk + C::BK - 1) / C::BK;
  const int64_t total = (int64_t)a.mtiles * a.nsplit * a.B * a.Hk * (C::SP ? 2 : 1);
  return a.nsplit > 1 ? launch(attn_dkv_kernel<T, DP, NW, RG, WK, true>, total, C::NT, C::LDS, a, st)
                      : launch(attn_dkv_kernel<T, DP, NW, RG, WK, false>, total, C::NT, C::LDS, a, st);
}
template <typename T, int DP, int NW, bool WK>
int run_dq(Args& a, hipStream_t st) {
  typedef Dq<T, DP, NW, WK> C;
  a.mtiles = (a.M + C::BM - 1) / C::BM;
  const int64_t total = (int64_t)a.mtiles * a.nsplit * a.B * a.Hk;
  return a.nsplit > 1 ? launch(attn_dq_kernel<T, DP, NW, WK, true>, total, C::NT, C::LDS, a, st)
                      : launch(attn_dq_kernel<T, DP, NW, WK, false>, total, C::NT, C::LDS, a, st);
}
template <typename T, int DP>
int bwd(Args& a, Shape kv, Shape q, float* part_kv, float* part_q, float* delta, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.Hq;
  attn_delta_kernel<T><<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(a, delta);
  int rc = (int)hipGetLastError();
  if (rc) return rc;
  a.delta = delta;
  constexpr int WK = sizeof(T) == 4 && DP == 128 ? 2 : 4;
  Sum sums[2] = {};
  if (a.dk) {
    a.nsplit = kv.split;
    a.part = part_kv;
    rc = kv.few ? run_dkv<T, DP, WK, 1, true>(a, st) : run_dkv<T, DP, 4, sizeof(T) == 2 && DP == 128 ? 2 : 1, false>(a, st);
    if (rc) return rc;
    if (kv.split > 1) sums[0] = Sum{part_kv, a.dk, a.dv, (int64_t)a.B * a.Sk * a.Hk * a.D, kv.split};
  }
  if (a.dq) {
    a.nsplit = q.split;
    a.part = part_q;
    rc = q.few ? run_dq<T, DP, WK, true>(a, st) : run_dq<T, DP, 4, false>(a, st);
    if (rc) return rc;
    if (q.split > 1) sums[1] = Sum{part_q, a.dq, nullptr, rows * a.D, q.split};
  }
  const int64_t most = std::max(2 * sums[0].n, sums[1].n);
  if (!most) return 0;
  attn_sum_kernel<T><<<dim3((unsigned)((most / 4 + 255) / 256), 2), 256, 0, st>>>(sums[0], sums[1]);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace turtle

using namespace turtle;

extern "C" {

size_t turtle_token_attn_bwd_workspace(const turtle_token_attn_args* x, int dtype) {
  if (!sizes_ok(x, dtype) || x->table) return 0;
  return part_bytes(x, dtype, false) + part_bytes(x, dtype, true);
}

int turtle_token_attn_bwd(const turtle_token_attn_grads* g, int dtype, void* stream) {
  Args a;
  if (!g || g->f.table || !fill(a, &g->f, dtype)) return -1;
  const int es = dtype == 0 ? 4 : 2;
  if (!rows16(g->dout, g->gb, g->gs, g->gh, es) || !a.lse || (!g->dk) != (!g->dv) || !g->delta) return -1;
  const size_t n = turtle_token_attn_bwd_workspace(&g->f, dtype);
  if (n && (!g->f.ws || g->f.ws_bytes < n || (uintptr_t)g->f.ws % 16)) return -1;
  const Shape kv = shape_of(&g->f, dtype, false), q = shape_of(&g->f, dtype, true);
  float *pkv = (float*)g->f.ws, *pq = pkv + part_bytes(&g->f, dtype, false) / sizeof(float);
  a.dout = g->dout; a.gb = g->gb; a.gs = g->gs; a.gh = g->gh;
  a.dq = g->dq; a.dk = g->dk; a.dv = g->dv;
  hipStream_t st = (hipStream_t)stream;
  const bool small = a.D <= 64;
  if (dtype == 0) return small ? bwd<float, 64>(a, kv, q, pkv, pq, g->delta, st) : bwd<float, 128>(a, kv, q, pkv, pq, g->delta, st);
  if (dtype == 1) return small ? bwd<bf16, 64>(a, kv, q, pkv, pq, g->delta, st) : bwd<bf16, 128>(a, kv, q, pkv, pq, g->delta, st);
  return small ? bwd<f16, 64>(a, kv, q, pkv, pq, g->delta, st) : bwd<f16, 128>(a, kv, q, pkv, pq, g->delta, st);
}

}  // extern "C"
