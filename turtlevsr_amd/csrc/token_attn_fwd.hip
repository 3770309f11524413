// Token attention, forward: dense and paged (token_attn.h holds the method and the shared parts).
//
// Three shapes of one kernel, chosen in plan_of by the rows M = Sq G of a (sequence, key head) and the keys:
//   kind 0   the block's waves take the key tiles of 32 rows in turn, each with its own LDS ring and no block barrier, and
//            join at the end
//   kind 1   2 waves x 32 rows
//   kind 2   4 waves x 32 rows
// The first two have matrix instructions to spare and multiply p in two terms (TWO): with few keys, p's rounding
// would be as large an error as the result's own.
//
// Measured: 32640 x 32640 tokens, 8 heads of 64 channels, bf16, 2450 - 2700 us (810 - 890 TF/s; at 64 rows a wave instead of 32, no
// faster: 2 x 16 more registers hold off one of three waves of a SIMD); causal with prefix 2048, 2 x 5120 tokens, 108 us
// (575 TF/s); 510 windows of 64 tokens, 4 heads, 19 us (3.5 TB/s; the start of its one-tile blocks); one token on 16
// histories of up to 16384 keys, 16 heads on 4 of 128 channels, 80 + 5 us for the join (4.5 TB/s while it reads); 256
// tokens on 4 histories of 5040, fp16, 8 heads, 32 + 6 us.
#include "token_attn.h"

namespace turtle {
namespace {

template <typename T, int DP, int NW, bool WK> struct Fwd {
  typedef Rows<T, DP> R;
  static constexpr int NT = NW * 64;
  static constexpr int BM = WK ? 32 : NW * 32;        // rows of a block, 32 a wave
  static constexpr int BN = (WK || sizeof(T) == 4) ? 32 : 64;
  static constexpr int NS = 2;                        // slots of the ring
  static constexpr int TILE = BN * R::ROWB, SLOT = 2 * TILE + 512;      // K, V; document of a key
  static constexpr int LT = WK ? 64 : NT;             // threads that load a tile
  static constexpr int NLD = R::template loads2<BN, LT>();
  static constexpr int WIN = 256;                     // page numbers a wave keeps at hand
  static constexpr bool TWO = sizeof(T) == 2 && (WK || NW == 2);
  // the tile's probabilities as operands of the second product
  struct P {
    uint4 hi[2 * BN / 32], lo[TWO ? 2 * BN / 32 : 1];
    float x[sizeof(T) == 4 ? 2 * BN / 32 : 1][8];
    // 8 values; returns l + their sum (16-bit types: of what the product takes)
    TURTLE_DEV float put(int u, const float (&v)[8], float l) {
      if constexpr (sizeof(T) == 2) {
        hi[u] = R::pack(v);
        if constexpr (!TWO) return R::sum_packed(hi[u], l);
        else lo[u] = R::rest(v, hi[u]);
      }
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        a += v[e]; b += v[e + 1];
        if constexpr (sizeof(T) == 4) { x[u][e] = v[e]; x[u][e + 1] = v[e + 1]; }
      }
      return l + (a + b);
    }
    template <int U> TURTLE_DEV void times(const char* vt, f32x16 (&acc)[R::DT], int lane) const {
      if constexpr (sizeof(T) == 2) R::template t_times<U, TWO>(vt, hi[U], lo[TWO ? U : 0], acc, lane);
      else R::template t_times<U>(vt, x[U], acc, lane);
    }
  };
  // LDS without the page numbers; a call with fewer tiles than slots takes only those
  static int lds(int64_t keys) {
    const int64_t tiles = (keys + BN - 1) / BN;
    if (!WK) return SLOT * (int)(tiles < NS ? tiles : NS);
    const int buf = NW * NS * SLOT, join = (2 * NW * 32 + R::DT * 16 * 64) * 4;
    return buf > join ? buf : join;
  }
};

template <typename T, int DP, int NW, bool WK, bool PAGED>
__global__ __launch_bounds__(NW * 64, DP == 128 && sizeof(T) == 4 ? 1 : 2) void attn_fwd_kernel(Args a) {
  typedef Fwd<T, DP, NW, WK> F;
  typedef Rows<T, DP> R;
  constexpr int BN = F::BN, KT = BN / 32, DT = R::DT, STEP = WK ? NW : 1;
  // fp16: p is scaled by 2^6 (p of many keys would lose bits below the type's normal range) and stays under its 2^16
  constexpr float POFF = std::is_same<T, f16>::value ? 6.f : 0.f;
  constexpr float SLACK = 8.f;
  extern __shared__ __attribute__((aligned(512))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

  const int item = xcd_item(a);
  if (item >= a.total) return;
  const int mt = a.mtiles - 1 - item % a.mtiles, rest = item / a.mtiles;   // causal: the longest tiles first
  const int sp = rest % a.nsplit, bh = rest / a.nsplit, b = bh / a.Hk, hk = bh - b * a.Hk;

  int kn = a.Sk, nq = a.Sq, off = a.Sk - a.Sq;
  if constexpr (PAGED) {
    const int64_t room = (int64_t)a.page * a.maxpages;
    const int kl = a.kv_lens[b];
    nq = a.q_lens ? min(max(a.q_lens[b], 0), a.Sq) : a.Sq;
    off = kl - nq;
    kn = max(0, (int)min((int64_t)kl, room));
  }
  const int m0 = mt * F::BM, mend = min(a.M, nq * a.G), m1 = min(m0 + F::BM, mend);   // rows of this block that exist: [m0, m1)
  const int pre = (!PAGED && a.prefix) ? max(a.prefix[b], 0) : 0;
  const int mw = m0 + (WK ? 0 : wave * 32), mw1 = min(mw + 32, mend);     // ... of this wave
  const int mrow = mw + (lane & 31);
  Row row = row_of(a, b, hk, mrow, off, nq);

  // key tiles this block walks over
  int kend = kn;
  if (a.causal) kend = min(kn, max((m1 - 1) / a.G + off + 1, pre));
  if (m1 <= m0) kend = 0;
  int t1 = (max(kend, 0) + BN - 1) / BN, t0 = 0;
  if (a.nsplit > 1) {
    const int per = (t1 + a.nsplit - 1) / a.nsplit;
    t0 = min(t1, sp * per);
    t1 = min(t1, t0 + per);
  }
  DocWalk dw;
  dw.none();
  if (!PAGED && a.qdoc && m1 > m0) {
    dw.init(a.kr + (int64_t)b * a.nkr, a.nkr, doc_range(a.qr + (int64_t)b * a.nqr, a.nqr, m0 / a.G, (m1 - 1) / a.G + 1));
    dw.own_docs(row.on ? row.doc : -1);
  }
  // what this wave's rows see whole: keys before `whole`; and at all: keys before `some`
  const int whole = a.causal ? max(mw / a.G + off + 1, pre) : 0x7fffffff;
  const int some = mw1 <= mw ? 0 : (a.causal ? max((mw1 - 1) / a.G + off + 1, pre) : 0x7fffffff);

  uint4 qf[R::STEPS];
  const int qi = token_of(a, mrow), qg = mrow - qi * a.G;
  R::frag(row.on ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qb + (int64_t)qi * a.qs + (int64_t)(hk * a.G + qg) * a.qh : nullptr, a.D,
          qf, lane);

  char* buf = smem + (WK ? wave * F::NS * F::SLOT : 0);
  const char* kbase = reinterpret_cast<const char*>(a.k) + ((PAGED ? 0 : (int64_t)b * a.kb) + (int64_t)hk * a.kh) * R::ES;
  const char* vbase = reinterpret_cast<const char*>(a.v) + ((PAGED ? 0 : (int64_t)b * a.vb) + (int64_t)hk * a.vh) * R::ES;
  const int64_t kst = a.ks * R::ES, vst = a.vs * R::ES;
  const int ltid = WK ? lane : tid;
  typename R::template Lin<F::LT> klin, vlin;
  klin.init(ltid, kst);
  vlin.init(ltid, vst);
  // page numbers: this wave's window of the sequence's table, read from LDS - a global read per tile would have to
  // wait, in order, behind the tiles in flight
  int* win = reinterpret_cast<int*>(smem + a.lds_win) + wave * F::WIN;
  int wbase = 0, wend = 0;
  auto page_of = [&](int key) { return quot(key, a.page, a.pmul, a.psh); };
  // starts tile t's copy into dst; returns which of its keys are seen at all (bit = key within the tile)
  auto issue = [&](int t, char* dst) __attribute__((always_inline)) -> uint64_t {
    const int k0 = t * BN;
    if constexpr (PAGED) {
      const int p0 = page_of(k0), p1 = page_of(min(k0 + BN, kn) - 1);
      if (p0 < wbase || p1 >= wend) {
        wbase = p0;
        wend = p0 + F::WIN;
#pragma unroll
        for (int e = 0; e < F::WIN / 64; ++e) {
          const int p = p0 + e * 64 + lane;
          win[e * 64 + lane] = p < a.maxpages ? a.table[(int64_t)b * a.maxpages + p] : -1;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      const int in0 = k0 - p0 * a.page;
      if (in0 + BN <= a.page && k0 + BN <= kn && a.D == DP) {       // a whole tile of one page
        const int id = __builtin_amdgcn_readfirstlane(win[p0 - wbase]);
        if ((uint32_t)id < (uint32_t)a.npages) {
          klin.template load<BN>(dst, ltid, kbase + (int64_t)id * a.kb * R::ES + in0 * kst, kst);
          vlin.template load<BN>(dst + F::TILE, ltid, vbase + (int64_t)id * a.vb * R::ES + in0 * vst, vst);
          return ~0ull;
        }
      }
      R::template load2<BN, F::LT>(dst, dst + F::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
        const int key = k0 + r;
        if (key >= kn) return;
        const int pg = page_of(key), id = win[pg - wbase], in = key - pg * a.page;
        if ((uint32_t)id >= (uint32_t)a.npages) return;
        p0 = kbase + ((int64_t)id * a.kb + (int64_t)in * a.ks) * R::ES;
        p1 = vbase + ((int64_t)id * a.vb + (int64_t)in * a.vs) * R::ES;
      });
      const int key = k0 + (lane & (BN - 1));
      bool ok = key < kn;
      if (ok) ok = (uint32_t)win[page_of(key) - wbase] < (uint32_t)a.npages;
      return __ballot(ok);
    } else {
      const bool holes = dw.holes;
      if (dw.mixed) key_docs<BN>(a, b, k0, dst + 2 * F::TILE, lane);
      if (!holes && k0 + BN <= kn && a.D == DP) {
        klin.template load<BN>(dst, ltid, kbase + k0 * kst, kst);
        vlin.template load<BN>(dst + F::TILE, ltid, vbase + k0 * vst, vst);
        return ~0ull;
      }
      R::template load2<BN, F::LT>(dst, dst + F::TILE, ltid, a.D, [&](int r, const char*& p0, const char*& p1) {
        const int key = k0 + r;
        if (key >= kn || (holes && a.kdoc[(int64_t)b * a.Sk + key] < 0)) return;
        p0 = kbase + (int64_t)key * a.ks * R::ES;
        p1 = vbase + (int64_t)key * a.vs * R::ES;
      });
      return ~0ull;
    }
  };

  f32x16 acc[DT];
  float mx = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = zero16();

  // The walk: tiles are started NS - 1 turns before they are computed on (q: the tiles in flight, oldest first). With a
  // block the turn's barrier frees the slot of the tile before; a wave of its own starts the next tile at once.
  constexpr int NS = F::NS;
  static_assert(NS == 2, "one tile in flight: the last one ends the walk");
  struct Tile { int t; bool mixed, mine; uint64_t seen; } q[NS - 1];
  int tnew = WK ? t0 + wave : t0, fly = 0, into = 0, slot = 0;
  auto start = [&]() __attribute__((always_inline)) {
    Tile x{dw.template next<BN>(tnew, t1, STEP, 1, a.Sk, lane), false, true, ~0ull};
    x.mixed = dw.mixed;
    x.mine = dw.mine;
    if (x.t < t1) { x.seen = issue(x.t, buf + into * F::SLOT); ++fly; }
    tnew = x.t + STEP;
    into = into + 1 == NS ? 0 : into + 1;
#pragma unroll
    for (int i = 0; i + 2 < NS; ++i) q[i] = q[i + 1];
    q[NS - 2] = x;
  };
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) start();
  if constexpr (WK || NW > 2) {      // kind 1 has a few tiles, nothing worth keeping in flight
    arrived(qf);
    arrived(row.doc);
    arrived(row.slope2);
  }
  for (;;) {
    const Tile cur = q[0];
    if (cur.t >= t1) break;
    if constexpr (!WK) {
      vm_wait_tiles<F::NLD, NS - 2>(fly - 1);
      lds_barrier();
    }
    if (tnew < t1) start();
    else q[0].t = t1;
    if constexpr (WK) vm_wait_tiles<F::NLD, NS - 1>(fly - 1);
    const char* kt = buf + slot * F::SLOT;
    const char* vt = kt + F::TILE;
    const int k0 = cur.t * BN;
    const bool mixed = cur.mixed;
    uint64_t seen = cur.seen;

    if (k0 < some && cur.mine) {
      f32x16 s[KT];
      R::template times<KT>(kt, qf, s, lane);
      // the rules that apply to this tile, each in a pass of its own (uniform branches)
      const bool caus = k0 + BN > whole;
      bool gaps = k0 + BN > kn;
      if constexpr (PAGED) gaps = BN == 32 ? (uint32_t)seen != ~0u : seen != ~0ull;
      float mul = a.scale2;
      if (a.cap > 0.f) {
        tanh_all<T, KT>(s, a.icap, a.cap);
        mul = a.cap2;
      }
      if (a.slopes || mul <= 0.f) {
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int at = row.pos - k0 - j * 32 - 4 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = fmaf(-row.slope2, fabsf((float)(at - acc_row(r))), s[j][r] * mul);
        }
        mul = 1.f;
      }
      if (caus) {
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const int last = max(row.pos, pre - 1) - k0 - j * 32 - 4 * h;      // the last key in sight
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = acc_row(r) <= last ? s[j][r] : -INFINITY;
        }
      }
      if (gaps) {
        if constexpr (!PAGED) seen = kn - k0 >= 64 ? ~0ull : (1ull << (kn - k0)) - 1;
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          const uint32_t bits = (uint32_t)(seen >> (j * 32)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] = (bits >> acc_row(r)) & 1 ? s[j][r] : -INFINITY;
        }
      }
      if (mixed) {
        const int* kd = reinterpret_cast<const int*>(kt + 2 * F::TILE) + 4 * h;
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int4 doc = *reinterpret_cast<const int4*>(kd + j * 32 + 8 * c);
            const int dc[4] = {doc.x, doc.y, doc.z, doc.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][4 * c + e] = dc[e] == row.doc ? s[j][4 * c + e] : -INFINITY;
          }
      }

      // p = 2^(s - mx) against the running reference mx, a maximum of earlier tiles: it serves as long as no score of a
      // lane is over it by more than SLACK. Only else are the row's halves compared and the accumulators rescaled.
      float tm = -INFINITY;
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) tm = fmaxf(tm, s[j][r]);
      if (__any(!(tm * mul <= mx + SLACK))) {
        const float mn = fmaxf(mx, half_max(tm) * mul);
        const float al = __builtin_amdgcn_exp2f(mx - (mn == -INFINITY ? 0.f : mn));
        mx = mn;
        l *= al;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= al;
      }
      typename F::P p;
      const float sh = POFF - (mx == -INFINITY ? 0.f : mx);
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + e], mul, sh));
        l = p.put(u, x, l);
      }
      static_for<2 * KT>([&](auto u) { p.template times<u()>(vt, acc, lane); });
    }
    if constexpr (WK) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    --fly;
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  l = half_sum(l);

  if constexpr (WK) {
    // join the waves: their (max, sum), then the rescaled accumulators summed through LDS in wave order
    float* ml = reinterpret_cast<float*>(smem);
    float* sum = ml + 2 * NW * 32;
    __syncthreads();
    if (h == 0) { ml[wave * 32 + lane] = mx; ml[(NW + wave) * 32 + lane] = l; }
    __syncthreads();
    float mall = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mall = fmaxf(mall, ml[w * 32 + (lane & 31)]);
    const float mb = mall == -INFINITY ? 0.f : mall;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) l += ml[(NW + w) * 32 + (lane & 31)] * __builtin_amdgcn_exp2f(ml[w * 32 + (lane & 31)] - mb);
    const float f = __builtin_amdgcn_exp2f(mx - mb);
    mx = mall;
    for (int w = 0; w < NW; ++w) {
      if (wave == w) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float* p = sum + (dt * 16 + r) * 64 + lane;
            *p = (w ? *p : 0.f) + acc[dt][r] * f;
          }
      }
      __syncthreads();
    }
    // every wave takes its share of the channels
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[dt][r] = sum[(dt * 16 + r) * 64 + lane];
  }

  if (mrow >= a.M) return;
  // a row that sees nothing: zeros, whatever the tile's values were; a sum that is not a number stays one
  const bool none = l == 0.f || !row.on;
  const float inv = none ? 0.f : 1.f / l, lse = none ? INFINITY : mx + log2f(l) - POFF;
  const bool first = (!WK || wave == 0) && h == 0;
  const int64_t pi = ((int64_t)sp * a.B * a.Hk + bh) * a.M + mrow;
  const int64_t oi = (((int64_t)b * a.Sq + qi) * a.Hq + hk * a.G + qg) * a.D;
  if (first && a.nsplit > 1) a.plse[pi] = lse;
  if (first && a.nsplit <= 1 && a.lse) a.lse[(int64_t)bh * a.M + mrow] = kept_sum(lse);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if (WK && dt % NW != wave) continue;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * h;
      if (d >= a.D) continue;
      float v[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = none ? 0.f : acc[dt][4 * q4 + e] * inv; lo[e] = v[e] - to_f((T)v[e]); }
      if (a.nsplit > 1) {
        *reinterpret_cast<float4*>(a.part + pi * a.D + d) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        R::put4(reinterpret_cast<T*>(a.o) + oi + d, v);
        if (a.olo) R::put4(reinterpret_cast<T*>(a.olo) + oi + d, lo);
      }
    }
  }
}

__global__ __launch_bounds__(256) void doc_range_kernel(const int* __restrict__ qdoc, const int* __restrict__ kdoc, int4* qr, int4* kr, int B,
                                                        int Sq, int Sk, int nqr, int nkr) {
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= B * (nqr + nkr)) return;
  const bool isq = w < B * nqr;
  const int u = isq ? w : w - B * nqr, n = isq ? nqr : nkr, S = isq ? Sq : Sk;
  const int b = u / n, t = u - b * n, i = t * RT + lane;
  const int d = i < S ? (isq ? qdoc : kdoc)[(int64_t)b * S + i] : -1;
  int lo = d < 0 ? 0x7fffffff : d, hi = d < 0 ? -1 : d;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o, 64)); hi = max(hi, __shfl_xor(hi, o, 64)); }
  const bool bad = __any(i < S && d < 0), whole = __all(i >= S || d >= 0);
  if (lane == 0) (isq ? qr : kr)[(int64_t)b * n + t] = make_int4(lo, hi, whole && lo == hi ? 1 : 0, bad ? 1 : 0);
}

// results of the splits -> o: 4 channels a thread
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(Args a) {
  const int c4 = a.D / 4;
  const int64_t n = (int64_t)a.B * a.Hk * a.M, stride = n;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= n * c4) return;
  const int64_t r = u / c4;
  const int d = (int)(u - r * c4) * 4;
  float mx = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) {
    const float x = a.plse[s * stride + r];
    mx = fmaxf(mx, x == INFINITY ? -INFINITY : x);
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) {                    // unrolled, no branch: the loads of 8 splits are in flight
    const float x = a.plse[s * stride + r];
    const float4 p = *reinterpret_cast<const float4*>(a.part + (s * stride + r) * a.D + d);
    const bool none = x == INFINITY;
    const float w = none ? 0.f : __builtin_amdgcn_exp2f(x - mx);
    l += w;
    v[0] = fmaf(w, none ? 0.f : p.x, v[0]); v[1] = fmaf(w, none ? 0.f : p.y, v[1]);
    v[2] = fmaf(w, none ? 0.f : p.z, v[2]); v[3] = fmaf(w, none ? 0.f : p.w, v[3]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float lo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[e] *= inv; lo[e] = v[e] - to_f((T)v[e]); }
  const int64_t bh = r / a.M, m = r - bh * a.M, b = bh / a.Hk, hk = bh - b * a.Hk, i = m / a.G, g = m - i * a.G;
  const int64_t oi = ((b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D + d;
  Rows<T, 64>::put4(reinterpret_cast<T*>(a.o) + oi, v);
  if (a.olo) Rows<T, 64>::put4(reinterpret_cast<T*>(a.olo) + oi, lo);
  if (a.lse && d == 0) a.lse[r] = kept_sum(l == 0.f ? INFINITY : mx + log2f(l));
}

struct Plan { int kind, nsplit; int64_t mtiles; };      // kind: 0 waves split the keys, 1 two waves, 2 four waves

// The shape of the grid. All times are of bf16 and 64 / 128 channels, fp32 where its choice differs.
//   kind 0 gives four times the blocks of kind 2 and no barriers, but each block re-reads its keys for 32 rows only:
//   taken for up to 32 rows (24 rows x 1024 keys, 256 heads: 18 / 28 us for 24 / 32), and for small grids (1024 x 1024, 8
//   heads: 14 / 20 for 19 / 25; 32 heads: 32 / 67 for 23 / 32). A small grid with long keys has work enough when they
//   are split (256 rows x 4096 keys, 16 heads: 25 / 39 for 23 / 32; 2048 keys: 19 / 26 for 20 / 27). And with a tile or
//   less for each of the four waves there is nothing to split (24 x 24, 512 heads: 8 / 17 for 7 / 9; fp32, where only
//   kind 2 has no split and its blocks are large: 18 / 27 for 9 / 23 at 24 keys, but 25 for 34 at 64).
//   kind 1 is kind 2 with p in two terms, for few keys (256 x 256, 512 heads: 33 / 60 us, kind 2 25 / 39).
Plan plan_of(const In* x, int dtype) {
  const int64_t M = (int64_t)x->Sq * (x->Hq / x->Hk), bh = (int64_t)x->B * x->Hk, room = key_room(x);
  const bool half = dtype != 0;
  Plan p;
  int bm;
  const int64_t b64 = (M + 63) / 64 * bh, b128 = (M + 127) / 128 * bh;
  const bool small = b64 < 256 && (M <= 64 || b128 * room < (1 << 17));
  if ((M <= 32 || small) && room > (half ? 128 : 32)) { p.kind = 0; bm = 32; }
  else if (half && room <= 256) { p.kind = 1; bm = 64; }
  else { p.kind = 2; bm = 128; }
  p.mtiles = (M + bm - 1) / bm;
  // Too few blocks to fill the 256 CUs: the keys are split over blocks too, 512 at least each, and joined by a second
  // kernel. 16-bit types of up to 64 channels: two blocks a CU have room (256 rows x 8192 keys, 16 heads: 30 us, with one
  // 34); else one (one token, 16384 keys, 16 sequences x 4 key heads x 4, 128 channels: 92 us, with two 100).
  const int64_t full = half && x->D <= 64 ? 512 : 256;
  const int64_t blocks = p.mtiles * bh, want = blocks >= 256 ? 1 : full / blocks, most = std::max<int64_t>(1, room / 512);
  p.nsplit = (int)std::min<int64_t>({want, most, 64});
  return p;
}

size_t ranges_bytes(const In* x) {
  if (!x->qdoc) return 0;
  return (size_t)x->B * ((x->Sq + RT - 1) / RT + (x->Sk + RT - 1) / RT) * sizeof(int4);
}
size_t ws_bytes(const In* x, int dtype) {
  const Plan p = plan_of(x, dtype);
  if (p.nsplit <= 1) return 0;
  return (size_t)p.nsplit * x->B * x->Sq * x->Hq * (x->D + 1) * sizeof(float);
}

template <typename T, int DP, int NW, bool WK, bool PAGED>
int run(Args& a, const Plan& p, int64_t keys, hipStream_t st) {
  typedef Fwd<T, DP, NW, WK> F;
  a.lds_win = F::lds(keys);
  const int lds = a.lds_win + (PAGED ? NW * F::WIN * 4 : 0);
  return launch(attn_fwd_kernel<T, DP, NW, WK, PAGED>, p.mtiles * a.B * a.Hk * p.nsplit, F::NT, lds, a, st);
}

template <typename T, int DP, bool PAGED>
int fwd(Args& a, const Plan& p, int64_t keys, hipStream_t st) {
  constexpr int WK = sizeof(T) == 4 && DP == 128 ? 2 : 4;
  a.mtiles = (int)p.mtiles;
  a.nsplit = p.nsplit;
  int rc;
  if (p.kind == 0) rc = run<T, DP, WK, true, PAGED>(a, p, keys, st);
  else if (sizeof(T) == 2 && p.kind == 1) rc = run<T, DP, sizeof(T) == 4 ? 4 : 2, false, PAGED>(a, p, keys, st);
  else rc = run<T, DP, 4, false, PAGED>(a, p, keys, st);
  if (rc || p.nsplit <= 1) return rc;
  const int64_t n = (int64_t)a.B * a.Hk * a.M * (a.D / 4);
  attn_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  return (int)hipGetLastError();
}

template <typename T>
int fwd_any(Args& a, const Plan& p, int64_t keys, hipStream_t st) {
  const bool paged = a.table != nullptr;
  if (a.D <= 64) return paged ? fwd<T, 64, true>(a, p, keys, st) : fwd<T, 64, false>(a, p, keys, st);
  return paged ? fwd<T, 128, true>(a, p, keys, st) : fwd<T, 128, false>(a, p, keys, st);
}

}  // namespace
}  // namespace turtle

using namespace turtle;

extern "C" {

size_t turtle_token_attn_ranges(const turtle_token_attn_args* a) { return sizes_ok(a, 0) ? ranges_bytes(a) : 0; }
size_t turtle_token_attn_workspace(const turtle_token_attn_args* a, int dtype) { return sizes_ok(a, dtype) ? ws_bytes(a, dtype) : 0; }

int turtle_token_attn_fwd(const turtle_token_attn_args* x, int dtype, void* stream) {
  Args a;
  if (!fill(a, x, dtype)) return -1;
  const Plan p = plan_of(x, dtype);
  if (p.nsplit > 1) {
    if (!x->ws || x->ws_bytes < ws_bytes(x, dtype) || (uintptr_t)x->ws % 16) return -1;
    a.part = (float*)x->ws;
    a.plse = a.part + (size_t)p.nsplit * x->B * x->Sq * x->Hq * x->D;
  }
  hipStream_t st = (hipStream_t)stream;
  if (x->qdoc) {
    const int n = x->B * (a.nqr + a.nkr);
    doc_range_kernel<<<(n + 3) / 4, 256, 0, st>>>(x->qdoc, x->kdoc, (int4*)a.qr, (int4*)a.kr, x->B, x->Sq, x->Sk, a.nqr, a.nkr);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  if (dtype == 0) return fwd_any<float>(a, p, key_room(x), st);
  if (dtype == 1) return fwd_any<bf16>(a, p, key_room(x), st);
  return fwd_any<f16>(a, p, key_room(x), st);
}

}  // extern "C"
