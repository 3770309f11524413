// Token attention: capped, biased and masked softmax(q k^T) v over clips of tokens, its backward, and the same
// forward over a paged cache (include/turtle_token.h).
//
// Rows. The G = Hq / Hk query heads that share a key head are rows of ONE problem: row m = i G + g is query i of
// head hk G + g, so keys and values are read once for all of them and a single new token of 8 sharing heads still
// fills 8 of a wave's 32 columns.
//
// One pass, everything in registers. A wave owns 32 rows. It computes S^T = K Q^T with 32x32 matrix instructions
// (keys x rows): a lane then holds scores of ONE row (row = lane & 31), so the softmax's running maximum, sum and
// rescaling factor are one register each and the maximum over keys is in-lane but for one exchange with lane ^ 32.
// The probabilities leave the accumulator layout as the B operand of O^T = V^T P^T: 8 consecutive accumulator
// registers of a lane are the keys 16 s + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} (h = lane >> 5), and any order of
// the contraction is right as long as V^T is read in the same one - which is what the transposing LDS read gives in
// two 4-key pieces. Nothing is exchanged through memory between the two products.
//
// Tiles of BN keys of K and V go HBM -> LDS by LDS-DMA, two buffers, the next tile in flight behind the current
// one's products. LDS rows are not padded (the DMA writes lane-linear): 16-byte chunk c of row r sits at chunk
// c ^ swz(r), applied on the DMA's source address, so that both the row reads (K: 32 rows, one chunk) and the
// transposing reads (V: 4 rows, 4 chunks) touch distinct banks.
//
// Backward, two kernels and no atomics, so results do not depend on the launch's order:
//   dk, dv: a wave owns 32 keys and walks over the rows: S = Q K^T, dP = dO V^T (rows x keys, lane = key), then
//           dV^T += dO^T P and dK^T += Q^T dS with the same register-to-operand step as above;
//   dq:     a wave owns 32 rows and walks over the keys: S^T, dP^T (lane = row), dQ^T += K^T dS^T.
//   delta_i = do_i . o_i uses o with its rounding remainder (o_lo): a row whose few keys make dP - delta cancel
//   would otherwise get 16-bit noise as its gradient.
//
// What is rounded: p and dS to the inputs' type as operands of the second products (fp16: p times 2^10, so that
// 1 / 10^4 keeps its bits), results at the end; scores, maxima, sums and accumulators are fp32.
#include "common.h"
#include "../../include/turtle_token.h"

#include <algorithm>
#include <type_traits>

namespace turtle {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) char lds_char;

__device__ __attribute__((aligned(64))) uint4 g_zero_ta[4];   // source of rows and channels that are not there

constexpr float LOG2E = 1.4426950408889634f;
constexpr int RT = 64;            // tokens of a document-range tile

template <typename T> TURTLE_DEV f32x16 mma(uint4 a, uint4 b, f32x16 c);
template <> TURTLE_DEV f32x16 mma<bf16>(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> TURTLE_DEV f32x16 mma<f16>(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// fp32: a 16-byte chunk pair is 8 channels, contracted two at a time in the order (e, 4 + e)
template <> TURTLE_DEV f32x16 mma<float>(uint4 a, uint4 b, f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
}

// accumulator register r of a 32x32 tile: its row (0..31) is acc_row(r) + 4 (lane >> 5)
constexpr TURTLE_DEV int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

TURTLE_DEV f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// combine over lane ^ 32
TURTLE_DEV float half_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
TURTLE_DEV float half_sum(float v) { return v + __shfl_xor(v, 32, 64); }

TURTLE_DEV uint32_t lds_addr(const char* p) { return (uint32_t)(uintptr_t)(const lds_char*)p; }

// 64 lanes x 16 B -> LDS (see gemm9.hip): inline asm, because the compiler would drain a builtin DMA before every
// LDS read; waited for by vm_wait
TURTLE_DEV void dma16(const void* gp, uint32_t lds_wave_base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(gp), "s"(lds_wave_base) : "memory");
}
// at most N vector-memory operations of this wave still in flight
template <int N>
TURTLE_DEV void vm_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// all of this wave's LDS accesses done, then the block's barrier
TURTLE_DEV void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A tile of rows of DP channels (zero past D) in LDS
template <typename T, int DP>
struct Rows {
  static constexpr int ES = sizeof(T), ROWB = DP * ES, CH = ROWB / 16, STEPS = ROWB / 32;
  static constexpr int DT = DP / 32;
  // the chunk exchange of row r: bijective over 16 rows (row reads), and over 4 rows in steps of 4 chunks
  // (transposing reads); 128-byte rows alternate between the two halves of the banks by themselves
  TURTLE_DEV static int swz(int r) {
    if constexpr (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  // row r's 16-byte chunk c
  TURTLE_DEV static uint4 chunk(const char* t, int r, int c) { return *reinterpret_cast<const uint4*>(t + r * ROWB + ((c ^ swz(r)) << 4)); }
  // acc += (32 rows from r0)(channels) x frag: frag is the B operand's STEPS chunks
  TURTLE_DEV static f32x16 times(const char* t, int r0, const uint4 (&frag)[STEPS], int lane) {
    f32x16 acc = zero16();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) acc = mma<T>(chunk(t, r0 + (lane & 31), 2 * s + (lane >> 5)), frag[s], acc);
    return acc;
  }
  // acc[dt] += (rows r0 .. r0 + 15)^T (channels 32 dt ..) x p: p = 8 accumulator registers' values of those rows
  TURTLE_DEV static void t_times(const char* t, int r0, const float (&p)[8], f32x16 (&acc)[DT], int lane) {
    const int h = lane >> 5;
    if constexpr (ES == 2) {
      const uint4 pb = pack(p);
      const int li = lane & 15, row = r0 + 4 * h + (li >> 2), sub = ((lane >> 4) & 1) * 2 + ((li & 3) >> 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const char* a = t + row * ROWB + (((dt * 4 + sub) ^ swz(row)) << 4) + (li & 1) * 8;
        const char* b = t + (row + 8) * ROWB + (((dt * 4 + sub) ^ swz(row + 8)) << 4) + (li & 1) * 8;
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a));
        const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b));
        acc[dt] = mma<T>(make_uint4(x.x, x.y, y.x, y.y), pb, acc[dt]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = r0 + acc_row(e) + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const int d = dt * 32 + (lane & 31);
          const float v = *reinterpret_cast<const float*>(t + row * ROWB + (((d >> 2) ^ swz(row)) << 4) + (d & 3) * 4);
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[e], acc[dt], 0, 0, 0);
        }
      }
    }
  }
  TURTLE_DEV static uint4 pack(const float (&p)[8]) {
    typedef T tx8 __attribute__((ext_vector_type(8)));
    tx8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (T)p[i];
    if constexpr (ES == 2) return __builtin_bit_cast(uint4, o);
    else return make_uint4(0, 0, 0, 0);
  }
  // one global row as the B operand: this lane's STEPS chunks (zero when p is null or past D channels)
  TURTLE_DEV static void frag(const T* p, int D, uint4 (&f)[STEPS], int lane) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int d = (2 * s + (lane >> 5)) * (16 / ES);
      f[s] = (p && d < D) ? *reinterpret_cast<const uint4*>(p + d) : make_uint4(0, 0, 0, 0);
    }
  }
  // DMA of N rows by NT threads: src(r) = address of row r's first channel, or null
  template <int N, int NT, typename F>
  TURTLE_DEV static void load(char* t, int tid, int D, F src) {
    static_assert(N * CH % NT == 0, "whole DMA instructions");
    const uint32_t base = lds_addr(t) + (uint32_t)(tid & ~63) * 16;
#pragma unroll
    for (int i = 0; i < N * CH / NT; ++i) {
      const int ci = i * NT + tid, r = ci / CH, c = (ci % CH) ^ swz(r);
      const char* s = reinterpret_cast<const char*>(src(r));
      const void* g = (s && c * 16 < D * ES) ? (const void*)(s + c * 16) : (const void*)g_zero_ta;
      dma16(g, __builtin_amdgcn_readfirstlane(base + (uint32_t)i * NT * 16));
    }
  }
  template <int N, int NT> static constexpr int loads() { return N * CH / NT; }
  // 4 consecutive channels d0 .. d0 + 3 of a dense result row
  TURTLE_DEV static void put4(T* p, const float (&v)[4]) {
    if constexpr (ES == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else {
      typedef T tx4 __attribute__((ext_vector_type(4)));
      tx4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
      *reinterpret_cast<tx4*>(p) = o;
    }
  }
};

struct Args {
  const void *q, *k, *v;
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh;
  int B, Sq, Sk, Hq, Hk, G, D, M;         // M = Sq * G rows of a (sequence, key head)
  float scale, scale2, cap, icap, cap2;   // scale2 = scale log2 e; cap2 = cap log2 e; icap = scale / cap
  const float* slopes;
  const int *prefix, *qdoc, *kdoc;
  const int4 *qr, *kr;                    // document ranges of RT-token tiles
  int nqr, nkr;
  int causal;
  int page, npages, maxpages;
  uint32_t pmul, psh;                     // j / page = mulhi(j, pmul) >> psh (page > 1)
  const int *table, *kv_lens, *q_lens;
  void *o, *olo;
  float* lse;
  int mtiles, nsplit, total;
  float *part, *plse;                     // [nsplit][B Hk][M][D], [nsplit][B Hk][M]
  // backward
  const void* dout;
  int64_t gb, gs, gh;
  void *dq, *dk, *dv;
  const float* delta;
};

// work item of a block: consecutive items on one XCD (blocks are dealt to the 8 XCDs in turn), so that the tiles
// of one key head share an L2
TURTLE_DEV int xcd_item(int total) {
  const int chunk = (total + 7) >> 3;
  const int i = (int)(blockIdx.x >> 3);
  return i < chunk ? (int)(blockIdx.x & 7) * chunk + i : total;
}

// One row's (query's) place and rules, in the lane that owns it
struct Row {
  int pos;       // its place among the keys; INT_MIN / 2 for no row
  int doc;
  float slope2;
  bool on;
};

TURTLE_DEV Row row_of(const Args& a, int b, int hk, int m, int off, int nq) {
  Row r;
  const int i = m / a.G, g = m - i * a.G;
  r.on = m < a.M && i < nq;
  r.pos = i + off;
  r.doc = (a.qdoc && r.on) ? a.qdoc[(int64_t)b * a.Sq + i] : 0;
  if (r.doc < 0) r.on = false;
  r.slope2 = (a.slopes && r.on) ? a.slopes[hk * a.G + g] * LOG2E : 0.f;
  return r;
}

// tanh for the cap. 16-bit inputs: 1 - 2 / (e^2x + 1), absolute error ~1e-7, under the scores' own rounding there;
// fp32: the library's, which keeps its relative error for small x
template <typename T>
TURTLE_DEV float cap_tanh(float x) {
  if constexpr (sizeof(T) == 4) return tanhf(x);
  else return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * LOG2E * x));
}

// pages
TURTLE_DEV const char* paged_row(const Args& a, const void* pool, int64_t sb, int64_t ss, int es, int b, int key, int64_t head) {
  const int pg = a.page == 1 ? key : (int)(__umulhi((uint32_t)key, a.pmul) >> a.psh);
  const int id = a.table[(int64_t)b * a.maxpages + pg];
  if ((uint32_t)id >= (uint32_t)a.npages) return nullptr;
  return reinterpret_cast<const char*>(pool) + ((int64_t)id * sb + (int64_t)(key - pg * a.page) * ss + head) * es;
}
TURTLE_DEV bool paged_seen(const Args& a, int b, int key) {
  const int pg = a.page == 1 ? key : (int)(__umulhi((uint32_t)key, a.pmul) >> a.psh);
  return (uint32_t)a.table[(int64_t)b * a.maxpages + pg] < (uint32_t)a.npages;
}

// Documents: the tiles of a walk that hold any number of [lo, hi], 64 tiles at a time. `ranges` of this sequence.
struct DocWalk {
  uint64_t mask;
  int base;
  // first tile >= t (of `ntile` in units of UNIT tokens) that may hold a visible token, or `end`
  template <int UNIT>
  TURTLE_DEV int next(int t, int end, const int4* ranges, int nr, int lo, int hi, int lane) {
    while (t < end) {
      if (base < 0 || t >= base + 64) {
        base = t;
        const int tt = t + lane;
        bool hit = false;
        if (tt < end) {
          for (int r = tt * UNIT / RT; r <= ((tt + 1) * UNIT - 1) / RT && r < nr; ++r) hit = hit || (ranges[r].x <= hi && ranges[r].y >= lo);
        }
        mask = __ballot(hit);
      }
      const uint64_t left = mask >> (t - base);
      if (left) return t + __builtin_ctzll(left);
      t = base + 64;
    }
    return end;
  }
};

// document range of tokens [t0, t1): {lo, hi, 1 if all are the same valid number, 1 if any is invalid}
TURTLE_DEV int4 doc_range(const int4* ranges, int nr, int t0, int t1) {
  int4 x = make_int4(0x7fffffff, -1, 1, 0);
  for (int r = t0 / RT; r <= (t1 - 1) / RT && r < nr; ++r) {
    const int4 y = ranges[r];
    x.x = min(x.x, y.x); x.y = max(x.y, y.y); x.z &= y.z; x.w |= y.w;
  }
  if (x.x != x.y) x.z = 0;
  return x;
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

// -------------------------------------------------------------------------------------------------
// forward
// -------------------------------------------------------------------------------------------------
// WK = 0: 4 waves x 32 rows share every key tile (block barriers). WK > 0: for at most 32 rows - WK waves take
// the key tiles in turn, each with its own buffers (no barriers), and join their results at the end.
template <typename T, int DP, int WK> struct Fwd {
  typedef Rows<T, DP> R;
  static constexpr int NW = WK ? WK : 4, NT = NW * 64;
  static constexpr int BM = WK ? 32 : 128;
  static constexpr int BN = (WK || sizeof(T) == 4) ? 32 : 64;
  static constexpr int TILE = BN * R::ROWB;
  static constexpr int LDS = 4 * TILE * (WK ? WK : 1);
  static constexpr int LT = WK ? 64 : NT;             // threads that load one tile
  static constexpr int NLD = 2 * (BN * R::CH / LT);   // DMA instructions of a K + V tile per thread
};

template <typename T, int DP, int WK, bool PAGED>
__global__ __launch_bounds__(WK ? WK * 64 : 256) void attn_fwd_kernel(Args a) {
  typedef Fwd<T, DP, WK> F;
  typedef Rows<T, DP> R;
  constexpr int BN = F::BN, KT = BN / 32, DT = R::DT;
  constexpr float POFF = std::is_same<T, f16>::value ? 10.f : 0.f;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;

  const int item = xcd_item(a.total);
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
  const int m0 = mt * F::BM, m1 = min(m0 + F::BM, min(a.M, nq * a.G));     // rows of this block that exist: [m0, m1)
  const int mrow = m0 + (WK ? 0 : wave * 32) + (lane & 31);
  const Row row = row_of(a, b, hk, mrow, off, nq);
  const int pre = (!PAGED && a.prefix) ? a.prefix[b] : 0;

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
  const int4* kr = nullptr;
  int4 qrange = make_int4(0, 0, 1, 0);
  if (!PAGED && a.qdoc && m1 > m0) {
    kr = a.kr + (int64_t)b * a.nkr;
    qrange = doc_range(a.qr + (int64_t)b * a.nqr, a.nqr, m0 / a.G, (m1 - 1) / a.G + 1);
  }
  DocWalk dw{0, -1};
  auto next = [&](int t) {
    if (!kr) return min(t, t1);
    if constexpr (WK > 0) {        // a wave keeps to its own turn of the tiles
      for (; t < t1; t += WK) {
        const int4 x = doc_range(kr, a.nkr, t * BN, t * BN + BN);
        if (x.x <= qrange.y && x.y >= qrange.x) break;
      }
      return min(t, t1);
    } else {
      return dw.next<BN>(t, t1, kr, a.nkr, qrange.x, qrange.y, lane);
    }
  };

  uint4 qf[R::STEPS];
  {
    const int i = mrow / a.G, g = mrow - i * a.G;
    const T* p = row.on ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qb + (int64_t)i * a.qs + (int64_t)(hk * a.G + g) * a.qh : nullptr;
    R::frag(p, a.D, qf, lane);
  }

  char* buf = smem + (WK ? wave * 4 * F::TILE : 0);
  const int ltid = WK ? lane : tid;
  auto issue = [&](int t, char* dst) {
    const bool holes = kr && doc_range(kr, a.nkr, t * BN, t * BN + BN).w;
    auto src = [&](const void* base, int64_t sb, int64_t ss, int64_t sh, int r) -> const char* {
      const int key = t * BN + r;
      if (key >= kn) return nullptr;
      if constexpr (PAGED) return paged_row(a, base, sb, ss, R::ES, b, key, hk * sh);
      if (holes && a.kdoc[(int64_t)b * a.Sk + key] < 0) return nullptr;
      return reinterpret_cast<const char*>(base) + ((int64_t)b * sb + (int64_t)key * ss + hk * sh) * R::ES;
    };
    R::template load<BN, F::LT>(dst, ltid, a.D, [&](int r) { return src(a.k, a.kb, a.ks, a.kh, r); });
    R::template load<BN, F::LT>(dst + F::TILE, ltid, a.D, [&](int r) { return src(a.v, a.vb, a.vs, a.vh, r); });
  };

  f32x16 acc[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) acc[i] = zero16();
  float mx = -INFINITY, l = 0.f;

  int t = next(WK ? t0 + wave : t0), par = 0;
  if (t < t1) issue(t, buf);
  while (t < t1) {
    const int tn = next(t + (WK ? WK : 1));
    if (tn < t1) {
      issue(tn, buf + (par ^ 1) * 2 * F::TILE);
      vm_wait<F::NLD>();
    } else {
      vm_wait<0>();
    }
    if constexpr (!WK) lds_barrier();
    const char* kt = buf + par * 2 * F::TILE;
    const char* vt = kt + F::TILE;

    f32x16 s[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) s[j] = R::times(kt, j * 32, qf, lane);

    // rules of this tile
    const int k0 = t * BN;
    bool docs = false;
    if (kr) {
      const int4 x = doc_range(kr, a.nkr, k0, k0 + BN);
      docs = !(x.z && qrange.z && x.x == qrange.x);
    }
    const bool caus = a.causal && k0 + BN > m0 / a.G + off + 1 && k0 + BN > pre;
    const bool masked = docs || caus || k0 + BN > kn || PAGED;
    float mul = a.scale2;
    if (masked || a.cap > 0.f || a.slopes || a.scale2 <= 0.f) {
      mul = 1.f;
      int kd = 0;
      if (docs) { const int key = k0 + (lane & (BN - 1)); kd = key < kn ? a.kdoc[(int64_t)b * a.Sk + key] : -1; }
      uint64_t seen = ~0ull;
      if constexpr (PAGED) { const int key = k0 + (lane & (BN - 1)); seen = __ballot(key < kn && paged_seen(a, b, key)); }
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kk = j * 32 + acc_row(r) + 4 * h, key = k0 + kk;
          float x = s[j][r];
          x = a.cap > 0.f ? a.cap2 * cap_tanh<T>(x * a.icap) : x * a.scale2;
          if (a.slopes) x -= row.slope2 * fabsf((float)(row.pos - key));
          if (masked) {
            bool vis = key < kn;
            if (docs) { const int d = __shfl(kd, kk, 64); vis = vis && d == row.doc; }   // every lane gives its number
            if (caus) vis = vis && (key <= row.pos || key < pre);
            if constexpr (PAGED) vis = vis && ((seen >> kk) & 1);
            x = vis ? x : -INFINITY;
          }
          s[j][r] = x;
        }
    }

    float tm = -INFINITY;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) tm = fmaxf(tm, s[j][r]);
    const float mn = fmaxf(mx, half_max(tm) * mul);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float al = __builtin_amdgcn_exp2f(mx - ms);
    mx = mn;
    float ls = 0.f;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[j][r], mul, POFF - ms));
        s[j][r] = p;
        ls += p;
      }
    l = fmaf(l, al, ls);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= al;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = s[j][8 * u + e];
        R::t_times(vt, j * 32 + u * 16, p, acc, lane);
      }
    if constexpr (!WK) lds_barrier();
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    par ^= 1;
    t = tn;
  }
  l = half_sum(l);

  if constexpr (WK > 0) {
    // join the waves: their (max, sum), then the rescaled accumulators summed through LDS in wave order
    float* ml = reinterpret_cast<float*>(smem);
    float* sum = ml + 2 * WK * 32;
    __syncthreads();
    if (h == 0) { ml[wave * 32 + lane] = mx; ml[(WK + wave) * 32 + lane] = l; }
    __syncthreads();
    float mall = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) mall = fmaxf(mall, ml[w * 32 + (lane & 31)]);
    const float mb = mall == -INFINITY ? 0.f : mall;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) l += ml[(WK + w) * 32 + (lane & 31)] * __builtin_amdgcn_exp2f(ml[w * 32 + (lane & 31)] - mb);
    const float f = __builtin_amdgcn_exp2f(mx - mb);
    for (int w = 0; w < WK; ++w) {
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
    mx = mall;
    // every wave takes its share of the channels
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[dt][r] = sum[(dt * 16 + r) * 64 + lane];
  }

  if (mrow >= a.M) return;
  const float inv = (l > 0.f && row.on) ? 1.f / l : 0.f;
  const float lse = inv > 0.f ? mx + log2f(l) - POFF : INFINITY;
  const int64_t mi = (int64_t)bh * a.M + mrow;
  const int i = mrow / a.G, g = mrow - i * a.G;
  const bool first = !WK || wave == 0;
  if (a.nsplit > 1) {
    const int64_t pi = ((int64_t)sp * a.B * a.Hk + bh) * a.M + mrow;
    if (first && h == 0) a.plse[pi] = lse;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (WK && dt % (WK ? WK : 1) != wave) continue;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d = dt * 32 + 8 * q4 + 4 * h;
        if (d < a.D)
          *reinterpret_cast<float4*>(a.part + pi * a.D + d) =
              make_float4(acc[dt][4 * q4] * inv, acc[dt][4 * q4 + 1] * inv, acc[dt][4 * q4 + 2] * inv, acc[dt][4 * q4 + 3] * inv);
      }
    }
    return;
  }
  if (first && h == 0 && a.lse) a.lse[mi] = lse;
  const int64_t oi = (((int64_t)b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if (WK && dt % (WK ? WK : 1) != wave) continue;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * h;
      if (d >= a.D) continue;
      float v[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = acc[dt][4 * q4 + e] * inv; lo[e] = v[e] - to_f((T)v[e]); }
      R::put4(reinterpret_cast<T*>(a.o) + oi + d, v);
      if (a.olo) R::put4(reinterpret_cast<T*>(a.olo) + oi + d, lo);
    }
  }
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
  for (int s = 0; s < a.nsplit; ++s) {
    const float x = a.plse[s * stride + r];
    if (x != INFINITY) mx = fmaxf(mx, x);
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float x = a.plse[s * stride + r];
    if (x == INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(x - mx);
    const float4 p = *reinterpret_cast<const float4*>(a.part + (s * stride + r) * a.D + d);
    l += w;
    v[0] = fmaf(w, p.x, v[0]); v[1] = fmaf(w, p.y, v[1]); v[2] = fmaf(w, p.z, v[2]); v[3] = fmaf(w, p.w, v[3]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  float lo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[e] *= inv; lo[e] = v[e] - to_f((T)v[e]); }
  const int64_t bh = r / a.M, m = r - bh * a.M, b = bh / a.Hk, hk = bh - b * a.Hk, i = m / a.G, g = m - i * a.G;
  const int64_t oi = ((b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D + d;
  Rows<T, 64>::put4(reinterpret_cast<T*>(a.o) + oi, v);
  if (a.olo) Rows<T, 64>::put4(reinterpret_cast<T*>(a.olo) + oi, lo);
  if (a.lse && d == 0) a.lse[r] = l > 0.f ? mx + log2f(l) : INFINITY;
}

// -------------------------------------------------------------------------------------------------
// backward
// -------------------------------------------------------------------------------------------------
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

// scores -> (p, dcap): p in the exponent's scale, of one pair. lse = +inf: 0
template <typename T>
TURTLE_DEV float pair_p(const Args& a, float raw, float slope2, int dist, float lse, bool vis, float& dcap) {
  float x;
  dcap = 1.f;
  if (a.cap > 0.f) { const float th = cap_tanh<T>(raw * a.icap); x = a.cap2 * th; dcap = 1.f - th * th; }
  else x = raw * a.scale2;
  if (a.slopes) x -= slope2 * fabsf((float)dist);
  return vis ? __builtin_amdgcn_exp2f(x - lse) : 0.f;
}

template <typename T, int DP> struct Bwd {
  typedef Rows<T, DP> R;
  static constexpr int BK = 128;                       // keys of a block (dk, dv): 4 waves x 32
  static constexpr int BM = 32;                        // rows of a tile
  static constexpr int TILE = BM * R::ROWB;
  static constexpr int INFO = BM * 20;                 // lse, delta, place, document, slope of each row
  static constexpr int LDS = 4 * TILE + 2 * INFO;
  static constexpr int NLD = 2 * (BM * R::CH / 256);
  // dq
  static constexpr int QM = 128, QN = 32;
  static constexpr int QTILE = QN * R::ROWB, QLDS = 4 * QTILE;
  static constexpr int QNLD = 2 * (QN * R::CH / 256);
};

template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dkv_kernel(Args a) {
  typedef Bwd<T, DP> C;
  typedef Rows<T, DP> R;
  constexpr int BM = C::BM, DT = R::DT;
  constexpr float POFF = std::is_same<T, f16>::value ? 10.f : 0.f, PS = std::is_same<T, f16>::value ? 1.f / 1024.f : 1.f;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int item = xcd_item(a.total);
  if (item >= a.total) return;
  const int kt = item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int k0 = kt * C::BK, k1 = min(k0 + C::BK, a.Sk), off = a.Sk - a.Sq;
  const int key = k0 + wave * 32 + (lane & 31);
  const int pre = a.prefix ? a.prefix[b] : 0;
  const int kdoc = (a.kdoc && key < a.Sk) ? a.kdoc[(int64_t)b * a.Sk + key] : 0;
  const bool kon = key < a.Sk && kdoc >= 0;

  uint4 kf[R::STEPS], vf[R::STEPS];
  R::frag(kon ? reinterpret_cast<const T*>(a.k) + (int64_t)b * a.kb + (int64_t)key * a.ks + (int64_t)hk * a.kh : nullptr, a.D, kf, lane);
  R::frag(kon ? reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vb + (int64_t)key * a.vs + (int64_t)hk * a.vh : nullptr, a.D, vf, lane);

  // rows that may see a key of this block
  int mfirst = 0;
  if (a.causal && k0 >= pre) mfirst = max(0, k0 - off) * a.G;
  const int t1 = (a.M + BM - 1) / BM, t0 = min(t1, mfirst / BM);
  const int4* qr = nullptr;
  int4 krange = make_int4(0, 0, 1, 0);
  if (a.qdoc) {
    qr = a.qr + (int64_t)b * a.nqr;
    krange = doc_range(a.kr + (int64_t)b * a.nkr, a.nkr, k0, k1);
  }
  auto next = [&](int t) {
    if (!qr) return min(t, t1);
    for (; t < t1; ++t) {
      const int4 x = doc_range(qr, a.nqr, t * BM / a.G, (min((t + 1) * BM, a.M) - 1) / a.G + 1);
      if (x.x <= krange.y && x.y >= krange.x) break;
    }
    return t;
  };
  float* info = reinterpret_cast<float*>(smem + 4 * C::TILE);
  struct Info { float lse, delta, slope2; int pos, doc; };
  auto fetch = [&](int t) {
    Info x{INFINITY, 0.f, 0.f, 0, -1};
    const int m = t * BM + tid;
    if (tid < BM && m < a.M) {
      const int64_t mi = (int64_t)bh * a.M + m;
      const Row r = row_of(a, b, hk, m, off, a.Sq);
      x.lse = a.lse[mi]; x.delta = a.delta[mi]; x.slope2 = r.slope2; x.pos = r.pos; x.doc = r.on ? r.doc : -1;
    }
    return x;
  };
  auto keep = [&](const Info& x, float* dst) {
    if (tid < BM) {
      dst[tid] = x.lse; dst[BM + tid] = x.delta; dst[2 * BM + tid] = x.slope2;
      reinterpret_cast<int*>(dst)[3 * BM + tid] = x.pos; reinterpret_cast<int*>(dst)[4 * BM + tid] = x.doc;
    }
  };
  auto issue = [&](int t, char* dst) {
    // rows that see nothing may hold anything: they are not read
    auto src = [&](const void* base, int64_t sb, int64_t ss, int64_t sh, int r) -> const char* {
      const int m = t * BM + r, i = m / a.G, g = m - i * a.G;
      if (m >= a.M || (a.causal && i + off < 0 && pre <= 0)) return nullptr;
      if (a.qdoc && a.qdoc[(int64_t)b * a.Sq + i] < 0) return nullptr;
      return reinterpret_cast<const char*>(base) + ((int64_t)b * sb + (int64_t)i * ss + (int64_t)(hk * a.G + g) * sh) * R::ES;
    };
    R::template load<BM, 256>(dst, tid, a.D, [&](int r) { return src(a.q, a.qb, a.qs, a.qh, r); });
    R::template load<BM, 256>(dst + C::TILE, tid, a.D, [&](int r) { return src(a.dout, a.gb, a.gs, a.gh, r); });
  };

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) { dk[i] = zero16(); dv[i] = zero16(); }

  int t = next(t0), par = 0;
  if (t < t1) {
    keep(fetch(t), info);
    issue(t, smem);
  }
  while (t < t1) {
    const int tn = next(t + 1);
    Info nx;
    if (tn < t1) {
      nx = fetch(tn);
      issue(tn, smem + (par ^ 1) * 2 * C::TILE);
      vm_wait<C::NLD>();
    } else {
      vm_wait<0>();
    }
    lds_barrier();
    const char* qt = smem + par * 2 * C::TILE;
    const char* gt = qt + C::TILE;
    const float* in = info + par * (C::INFO / 4);
    f32x16 s = R::times(qt, 0, kf, lane);
    f32x16 dp = R::times(gt, 0, vf, lane);

    const int m0 = t * BM, m1 = min(m0 + BM, a.M);
    const bool caus = a.causal && k1 > m0 / a.G + off + 1 && k1 > pre;
    bool docs = false;
    if (qr) {
      const int4 x = doc_range(qr, a.nqr, m0 / a.G, (m1 - 1) / a.G + 1);
      docs = !(x.z && krange.z && x.x == krange.x);
    }
    const bool special = docs || caus || a.cap > 0.f || a.slopes;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int rr = 8 * c + 4 * h;
      const float4 lse = *reinterpret_cast<const float4*>(in + rr), del = *reinterpret_cast<const float4*>(in + BM + rr);
      const float ls[4] = {lse.x, lse.y, lse.z, lse.w}, de[4] = {del.x, del.y, del.z, del.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * c + e;
        float p, dc = 1.f;
        bool vis = true;
        if (special) {
          const int pos = reinterpret_cast<const int*>(in)[3 * BM + rr + e];
          if (caus) vis = key <= pos || key < pre;
          if (docs) vis = vis && reinterpret_cast<const int*>(in)[4 * BM + rr + e] == kdoc;
          p = pair_p<T>(a, s[r], in[2 * BM + rr + e], pos - key, ls[e] - POFF, vis, dc);
        } else {
          p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, POFF - ls[e]));
        }
        s[r] = p;
        const float ds = p * ((dp[r] - de[e]) * (PS * dc));
        dp[r] = vis ? ds : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) { x[e] = s[8 * u + e]; y[e] = dp[8 * u + e]; }
      R::t_times(gt, u * 16, x, dv, lane);
      R::t_times(qt, u * 16, y, dk, lane);
    }
    if (tn < t1) keep(nx, info + (par ^ 1) * (C::INFO / 4));
    lds_barrier();
    par ^= 1;
    t = tn;
  }
  if (key >= a.Sk) return;
  const int64_t oi = (((int64_t)b * a.Sk + key) * a.Hk + hk) * a.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * h;
      if (d >= a.D) continue;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = kon ? dk[dt][4 * q4 + e] * a.scale : 0.f;
        y[e] = kon ? dv[dt][4 * q4 + e] * PS : 0.f;
      }
      R::put4(reinterpret_cast<T*>(a.dk) + oi + d, x);
      R::put4(reinterpret_cast<T*>(a.dv) + oi + d, y);
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dq_kernel(Args a) {
  typedef Bwd<T, DP> C;
  typedef Rows<T, DP> R;
  constexpr int BN = C::QN, DT = R::DT;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int item = xcd_item(a.total);
  if (item >= a.total) return;
  const int mt = a.mtiles - 1 - item % a.mtiles, bh = item / a.mtiles, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int off = a.Sk - a.Sq, m0 = mt * C::QM, m1 = min(m0 + C::QM, a.M);
  const int mrow = m0 + wave * 32 + (lane & 31);
  const Row row = row_of(a, b, hk, mrow, off, a.Sq);
  const int pre = a.prefix ? a.prefix[b] : 0;
  int kend = a.Sk;
  if (a.causal) kend = min(a.Sk, max((m1 - 1) / a.G + off + 1, pre));
  const int t1 = (max(kend, 0) + BN - 1) / BN;
  const int4* kr = nullptr;
  int4 qrange = make_int4(0, 0, 1, 0);
  if (a.qdoc) {
    kr = a.kr + (int64_t)b * a.nkr;
    qrange = doc_range(a.qr + (int64_t)b * a.nqr, a.nqr, m0 / a.G, (m1 - 1) / a.G + 1);
  }
  DocWalk dw{0, -1};
  auto next = [&](int t) { return kr ? dw.next<BN>(t, t1, kr, a.nkr, qrange.x, qrange.y, lane) : min(t, t1); };

  uint4 qf[R::STEPS], gf[R::STEPS];
  float lse = INFINITY, delta = 0.f;
  const int i = mrow / a.G, g = mrow - i * a.G;
  {
    const int hq = hk * a.G + g;
    R::frag(row.on ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qb + (int64_t)i * a.qs + (int64_t)hq * a.qh : nullptr, a.D, qf, lane);
    R::frag(row.on ? reinterpret_cast<const T*>(a.dout) + (int64_t)b * a.gb + (int64_t)i * a.gs + (int64_t)hq * a.gh : nullptr, a.D, gf, lane);
    if (row.on) { lse = a.lse[(int64_t)bh * a.M + mrow]; delta = a.delta[(int64_t)bh * a.M + mrow]; }
  }
  auto issue = [&](int t, char* dst) {
    const bool holes = kr && doc_range(kr, a.nkr, t * BN, t * BN + BN).w;
    auto src = [&](const void* base, int64_t sb, int64_t ss, int64_t sh, int r) -> const char* {
      const int key = t * BN + r;
      if (key >= a.Sk) return nullptr;
      if (holes && a.kdoc[(int64_t)b * a.Sk + key] < 0) return nullptr;
      return reinterpret_cast<const char*>(base) + ((int64_t)b * sb + (int64_t)key * ss + hk * sh) * R::ES;
    };
    R::template load<BN, 256>(dst, tid, a.D, [&](int r) { return src(a.k, a.kb, a.ks, a.kh, r); });
    R::template load<BN, 256>(dst + C::QTILE, tid, a.D, [&](int r) { return src(a.v, a.vb, a.vs, a.vh, r); });
  };
  f32x16 dq[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j) dq[j] = zero16();

  int t = next(0), par = 0;
  if (t < t1) issue(t, smem);
  while (t < t1) {
    const int tn = next(t + 1);
    if (tn < t1) {
      issue(tn, smem + (par ^ 1) * 2 * C::QTILE);
      vm_wait<C::QNLD>();
    } else {
      vm_wait<0>();
    }
    lds_barrier();
    const char* kt = smem + par * 2 * C::QTILE;
    const char* vt = kt + C::QTILE;
    f32x16 s = R::times(kt, 0, qf, lane);
    f32x16 dp = R::times(vt, 0, gf, lane);
    const int k0 = t * BN;
    bool docs = false;
    if (kr) {
      const int4 x = doc_range(kr, a.nkr, k0, k0 + BN);
      docs = !(x.z && qrange.z && x.x == qrange.x);
    }
    const bool caus = a.causal && k0 + BN > m0 / a.G + off + 1 && k0 + BN > pre;
    const bool masked = docs || caus || k0 + BN > a.Sk;
    if (masked || a.cap > 0.f || a.slopes) {
      int kd = 0;
      if (docs) { const int key = k0 + (lane & 31); kd = key < a.Sk ? a.kdoc[(int64_t)b * a.Sk + key] : -1; }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kk = acc_row(r) + 4 * h, key = k0 + kk;
        bool vis = key < a.Sk;
        if (docs) { const int d = __shfl(kd, kk, 64); vis = vis && d == row.doc; }
        if (caus) vis = vis && (key <= row.pos || key < pre);
        float dc;
        const float p = pair_p<T>(a, s[r], row.slope2, row.pos - key, lse, vis, dc);
        const float ds = p * ((dp[r] - delta) * dc);
        dp[r] = vis ? ds : 0.f;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -lse)) * (dp[r] - delta);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = dp[8 * u + e];
      R::t_times(kt, u * 16, x, dq, lane);
    }
    lds_barrier();
    par ^= 1;
    t = tn;
  }
  if (mrow >= a.M) return;
  const int64_t oi = (((int64_t)b * a.Sq + i) * a.Hq + hk * a.G + g) * a.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * h;
      if (d >= a.D) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = row.on ? dq[dt][4 * q4 + e] * a.scale : 0.f;
      R::put4(reinterpret_cast<T*>(a.dq) + oi + d, x);
    }
}

// -------------------------------------------------------------------------------------------------
// host
// -------------------------------------------------------------------------------------------------
typedef turtle_token_attn_args In;

bool rows16(const void* p, int64_t sb, int64_t ss, int64_t sh, int es) {
  return p && (uintptr_t)p % 16 == 0 && sb * es % 16 == 0 && ss * es % 16 == 0 && sh * es % 16 == 0;
}

bool sizes_ok(const In* x, int dtype) {
  if (!x || dtype < 0 || dtype > 2 || x->B <= 0 || x->Sq <= 0 || x->Hq <= 0 || x->Hk <= 0 || x->Hq % x->Hk) return false;
  if (x->D <= 0 || x->D % 8 || x->D > 128) return false;
  const int64_t G = x->Hq / x->Hk;
  if ((int64_t)x->Sq * G >= (1ll << 30) || (int64_t)x->B * x->Hk >= (1ll << 24)) return false;
  if (x->table) {
    if (x->page <= 0 || x->npages < 0 || x->maxpages <= 0 || (int64_t)x->page * x->maxpages >= (1ll << 30)) return false;
  } else if (x->Sk <= 0 || x->Sk >= (1 << 30)) {
    return false;
  }
  return true;
}

// keys that a sequence can have
int64_t key_room(const In* x) { return x->table ? (int64_t)x->page * x->maxpages : x->Sk; }

struct Plan { bool few; int bm, nsplit; int64_t mtiles; };

// At most 32 rows: the waves of a block split the keys. Too few blocks to fill the 256 CUs: the keys are split
// over blocks as well, in pieces of at least 4 tiles a wave, and a second kernel joins the pieces.
Plan plan_of(const In* x) {
  Plan p;
  const int64_t M = (int64_t)x->Sq * (x->Hq / x->Hk);
  p.few = M <= 32;
  p.bm = p.few ? 32 : 128;
  p.mtiles = (M + p.bm - 1) / p.bm;
  const int64_t blocks = p.mtiles * x->B * x->Hk, room = key_room(x);
  const int64_t want = std::max<int64_t>(1, 256 / blocks), most = std::max<int64_t>(1, room / 512);
  p.nsplit = (int)std::min<int64_t>({want, most, 64});
  return p;
}

size_t ranges_bytes(const In* x) {
  if (!x->qdoc) return 0;
  return (size_t)x->B * ((x->Sq + RT - 1) / RT + (x->Sk + RT - 1) / RT) * sizeof(int4);
}
size_t ws_bytes(const In* x) {
  const Plan p = plan_of(x);
  if (p.nsplit <= 1) return 0;
  return (size_t)p.nsplit * x->B * x->Sq * x->Hq * (x->D + 1) * sizeof(float);
}

bool fill(Args& a, const In* x, int dtype) {
  if (!sizes_ok(x, dtype)) return false;
  const int es = dtype == 0 ? 4 : 2;
  if (!rows16(x->q, x->qb, x->qs, x->qh, es) || !rows16(x->k, x->kb, x->ks, x->kh, es) || !rows16(x->v, x->vb, x->vs, x->vh, es)) return false;
  if (!x->o || (uintptr_t)x->o % 16 || (uintptr_t)x->o_lo % 16) return false;
  if (x->prefix && !x->causal) return false;
  if ((x->qdoc != nullptr) != (x->kdoc != nullptr)) return false;
  if (x->qdoc && !x->ranges) return false;
  if (x->table && (!x->kv_lens || x->qdoc || x->prefix)) return false;
  a = Args{};
  a.q = x->q; a.k = x->k; a.v = x->v;
  a.qb = x->qb; a.qs = x->qs; a.qh = x->qh; a.kb = x->kb; a.ks = x->ks; a.kh = x->kh; a.vb = x->vb; a.vs = x->vs; a.vh = x->vh;
  a.B = x->B; a.Sq = x->Sq; a.Sk = x->table ? 0 : x->Sk; a.Hq = x->Hq; a.Hk = x->Hk; a.G = x->Hq / x->Hk; a.D = x->D; a.M = x->Sq * a.G;
  a.scale = x->scale; a.scale2 = x->scale * LOG2E; a.cap = x->softcap;
  if (x->softcap > 0.f) { a.icap = x->scale / x->softcap; a.cap2 = x->softcap * LOG2E; }
  a.slopes = x->slopes; a.prefix = x->prefix; a.qdoc = x->qdoc; a.kdoc = x->kdoc; a.causal = x->causal;
  a.nqr = (x->Sq + RT - 1) / RT; a.nkr = x->table ? 0 : (x->Sk + RT - 1) / RT;
  a.qr = (const int4*)x->ranges; a.kr = a.qr ? a.qr + (int64_t)x->B * a.nqr : nullptr;
  a.page = x->page; a.npages = x->npages; a.maxpages = x->maxpages; a.table = x->table; a.kv_lens = x->kv_lens; a.q_lens = x->q_lens;
  if (x->table && x->page > 1) {
    // j / page for j < 2^30: with l = ceil(log2 page), floor(j m / 2^(31 + l)) for m = floor(2^(31 + l) / page) + 1 is exact
    int l = 0;
    while ((1ll << l) < x->page) ++l;
    a.pmul = (uint32_t)((1ull << (31 + l)) / (uint64_t)x->page + 1);
    a.psh = (uint32_t)(l - 1);
  }
  a.o = x->o; a.olo = dtype == 0 ? nullptr : x->o_lo; a.lse = x->lse;
  return true;
}

template <typename K>
int launch(K kernel, int64_t total, int threads, int lds, Args& a, hipStream_t st) {
  if (total <= 0 || total >= (1ll << 30)) return -1;
  a.total = (int)total;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
  }
  kernel<<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(threads), lds, st>>>(a);
  return (int)hipGetLastError();
}

template <typename T, int DP, bool PAGED>
int fwd(Args& a, const Plan& p, hipStream_t st) {
  constexpr int WK = sizeof(T) == 4 && DP == 128 ? 2 : 4;
  a.mtiles = (int)p.mtiles;
  a.nsplit = p.nsplit;
  const int64_t total = p.mtiles * a.B * a.Hk * p.nsplit;
  int rc;
  if (p.few) rc = launch(attn_fwd_kernel<T, DP, WK, PAGED>, total, Fwd<T, DP, WK>::NT, Fwd<T, DP, WK>::LDS, a, st);
  else rc = launch(attn_fwd_kernel<T, DP, 0, PAGED>, total, Fwd<T, DP, 0>::NT, Fwd<T, DP, 0>::LDS, a, st);
  if (rc || p.nsplit <= 1) return rc;
  const int64_t n = (int64_t)a.B * a.Hk * a.M * (a.D / 4);
  attn_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  return (int)hipGetLastError();
}

template <typename T>
int fwd_any(Args& a, const Plan& p, hipStream_t st) {
  const bool paged = a.table != nullptr;
  if (a.D <= 64) return paged ? fwd<T, 64, true>(a, p, st) : fwd<T, 64, false>(a, p, st);
  return paged ? fwd<T, 128, true>(a, p, st) : fwd<T, 128, false>(a, p, st);
}

template <typename T, int DP>
int bwd(Args& a, float* delta, hipStream_t st) {
  typedef Bwd<T, DP> C;
  const int64_t rows = (int64_t)a.B * a.Sq * a.Hq;
  attn_delta_kernel<T><<<(unsigned)((rows + 31) / 32), 256, 0, st>>>(a, delta);
  int rc = (int)hipGetLastError();
  if (rc) return rc;
  a.delta = delta;
  if (a.dk) {
    a.mtiles = (a.Sk + C::BK - 1) / C::BK;
    rc = launch(attn_dkv_kernel<T, DP>, (int64_t)a.mtiles * a.B * a.Hk, 256, C::LDS, a, st);
    if (rc) return rc;
  }
  if (!a.dq) return 0;
  a.mtiles = (a.M + C::QM - 1) / C::QM;
  return launch(attn_dq_kernel<T, DP>, (int64_t)a.mtiles * a.B * a.Hk, 256, C::QLDS, a, st);
}

}  // namespace
}  // namespace turtle

using namespace turtle;

extern "C" {

size_t turtle_token_attn_ranges(const turtle_token_attn_args* a) { return a ? ranges_bytes(a) : 0; }
size_t turtle_token_attn_workspace(const turtle_token_attn_args* a, int dtype) { return sizes_ok(a, dtype) ? ws_bytes(a) : 0; }

int turtle_token_attn_fwd(const turtle_token_attn_args* x, int dtype, void* stream) {
  Args a;
  if (!fill(a, x, dtype)) return -1;
  const Plan p = plan_of(x);
  if (p.nsplit > 1) {
    if (!x->ws || x->ws_bytes < ws_bytes(x) || (uintptr_t)x->ws % 16) return -1;
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
  if (dtype == 0) return fwd_any<float>(a, p, st);
  if (dtype == 1) return fwd_any<bf16>(a, p, st);
  return fwd_any<f16>(a, p, st);
}

int turtle_token_attn_bwd(const turtle_token_attn_grads* g, int dtype, void* stream) {
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

}  // extern "C"
