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
// Tiles of BN keys of K and V go HBM -> LDS by LDS-DMA into a ring of NS slots, NS - 1 tiles in flight behind the
// current one's products; one barrier a tile (it frees the slot of the tile before). LDS rows are not padded (the DMA
// writes lane-linear): 16-byte chunk c of row r sits at chunk c ^ swz(r), applied on the DMA's source address, so that
// both the row reads (K: 32 rows, one chunk) and the transposing reads (V: 4 rows, 4 chunks) touch distinct banks.
//
// Backward, two kernels and no atomics, so results do not depend on the launch's order:
//   dk, dv: a wave owns 32 keys and walks over the rows: S = Q K^T, dP = dO V^T (rows x keys, lane = key), then
//           dV^T += dO^T P and dK^T += Q^T dS with the same register-to-operand step as above;
//   dq:     a wave owns 32 rows and walks over the keys: S^T, dP^T (lane = row), dQ^T += K^T dS^T.
//   delta_i = do_i . o_i uses o with its rounding remainder (o_lo): a row whose few keys make dP - delta cancel
//   would otherwise get 16-bit noise as its gradient.
//
// What is rounded: p and dS to the inputs' type as operands of the second products (fp16: p times 2^6 in the forward,
// which leaves room for the 2^8 it may stand over the running maximum, 2^10 for dv, so that p of 10^4 keys keep their
// bits; dS times a power of two of the row's or key's own), results at the end; scores, maxima, sums and accumulators are
// fp32. The 16-bit rounding of p and dS is what separates the 16-bit results from the rounded exact ones: relative error of
// all values 2.4e-3 in bf16 and 3.0e-4 in fp16, the rounding of the result alone being 1.7e-3 and 2.1e-4.
// Where p has one term, the row's sum (in fp32) is of the rounded p, so that o's weights add up to one; the backward's p
// takes it too and is off, all of a row alike, by half a step at most (bf16: 1.5e-3 in rows of a few keys, 3e-4 at 1500).
//
// Bound: the matrix products where rows are many (a large bf16 product reaches 1188 TF/s on the card, fp32 153), HBM
// where they are few (a large copy reaches 4.9 TB/s). Beside the products every score costs an exponential (10 clocks of
// a SIMD, the 32 x 32 product of 16 channels 35) and about five more vector instructions, and every operand an LDS read.
#pragma once
#include "common.h"
#include "../../include/turtle_token.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>


namespace turtle {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_ __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_ __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
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
// LDS reads by address: 16 bytes, a float, and 4 x 16 elements of a group of 16 lanes transposed (a lane gives the place
// of 8 bytes and gets its column)
TURTLE_DEV uint4 lds_ld16(uint32_t a) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(uint4, *(__attribute__((address_space(3))) const u32x4*)a);
#else
  return make_uint4(a, 0, 0, 0);
#endif
}
TURTLE_DEV float lds_ld4(uint32_t a) {
#if defined(__HIP_DEVICE_COMPILE__)
  return *(__attribute__((address_space(3))) const float*)a;
#else
  return (float)a;
#endif
}
TURTLE_DEV uint2 lds_ld_tr(uint32_t a) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a));
#else
  return make_uint2(a, 0);
#endif
}

// 64 lanes x 16 B -> LDS (see gemm9.hip): inline asm, because the compiler would drain a builtin DMA before every
// LDS read; waited for by vm_wait
TURTLE_DEV void dma16(const void* gp, uint32_t lds_wave_base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(gp), "s"(lds_wave_base) : "memory");
}
// 64 lanes x 4 B -> LDS
TURTLE_DEV void dma4(const void* gp, uint32_t lds_wave_base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(gp), "s"(lds_wave_base) : "memory");
}
// at most N vector-memory operations of this wave still in flight
template <int N>
TURTLE_DEV void vm_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// at most N tiles of NLD operations each still in flight, N known at run time
template <int NLD, int MOST>
TURTLE_DEV void vm_wait_tiles(int n) {
  if constexpr (MOST <= 0) vm_wait<0>();
  else if (n >= MOST) vm_wait<NLD * MOST>();
  else vm_wait_tiles<NLD, MOST - 1>(n);
}
// all of this wave's LDS accesses done, then the block's barrier
TURTLE_DEV void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int N, typename F, int... I>
TURTLE_DEV void static_for_(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
TURTLE_DEV void static_for(F f) { static_for_<N>(f, std::make_integer_sequence<int, N>{}); }

// Values loaded before a loop are waited for here: left to their first use inside it, the wait would stand in the loop and
// drain the copies in flight at every turn
TURTLE_DEV void arrived(uint4& x) { asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w)); }
TURTLE_DEV void arrived(float& x) { asm volatile("" : "+v"(x)); }
TURTLE_DEV void arrived(int& x) { asm volatile("" : "+v"(x)); }
template <typename X, int N>
TURTLE_DEV void arrived(X (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) arrived(x[i]);
}

// N steps of an LDS read and a product: read n + AHEAD is started before product n, by the order that an empty statement
// with memory effects keeps. Left alone the compiler reads an operand right before its product and waits the read out
// each time (a wave alone on its SIMD has nothing else to do then).
template <int N, int AHEAD, typename Read, typename Use>
TURTLE_DEV void in_steps(Read read, Use use) {
  typedef decltype(read(std::integral_constant<int, 0>{})) V;
  V v[AHEAD + 1];
  static_for<(AHEAD < N ? AHEAD : N)>([&](auto n) { v[n()] = read(n); });
  static_for<N>([&](auto n) {
    if constexpr (n() + AHEAD < N) v[(n() + AHEAD) % (AHEAD + 1)] = read(std::integral_constant<int, n() + AHEAD>{});
    u32x4 x = __builtin_bit_cast(u32x4, v[n() % (AHEAD + 1)]);
    asm volatile("" : "+v"(x) : : "memory");
    use(n, __builtin_bit_cast(V, x));
  });
}

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
  // LDS addresses. A tile starts at a multiple of ROWB and swz(r + 16) = swz(r), swz(r + 8) = swz(r) ^ 2, so all of a
  // lane's addresses are one base with bits exchanged: no register per chunk.
  // this lane's place in row reads: row (lane & 31), chunk (lane >> 5); chunk 2 s + (lane >> 5) is at ^ (s << 5)
  TURTLE_DEV static uint32_t row_base(const char* t, int lane) {
    return lds_addr(t) + (lane & 31) * ROWB + (((lane >> 5) ^ swz(lane & 31)) << 4);
  }
  template <int S, int J> TURTLE_DEV static uint4 chunk(uint32_t base) { return lds_ld16((base ^ (S << 5)) + J * 32 * ROWB); }
  // ... in transposing reads of 16 rows: 4 rows from 4 (lane >> 5), 8 bytes of a chunk; channels 32 dt .. are at
  // ^ (dt << 6), the rows 8 further at ^ 32, + 8 ROWB
  TURTLE_DEV static uint32_t tr_base(const char* t, int lane) {
    const int li = lane & 15, row = 4 * (lane >> 5) + (li >> 2), sub = ((lane >> 4) & 1) * 2 + ((li & 3) >> 1);
    return lds_addr(t) + row * ROWB + ((sub ^ swz(row)) << 4) + (li & 1) * 8;
  }
  // acc[j] = (rows 32 j .. 32 j + 31)(channels) x frag, the KT chains of products interleaved: frag is the B operand's
  // STEPS chunks
  template <int KT>
  TURTLE_DEV static void times(const char* t, const uint4 (&frag)[STEPS], f32x16 (&acc)[KT], int lane) {
    const uint32_t base = row_base(t, lane);
#pragma unroll
    for (int j = 0; j < KT; ++j) acc[j] = zero16();
    in_steps<KT * STEPS, 3>([&](auto n) { return chunk<n() / KT, n() % KT>(base); },
                                 [&](auto n, uint4 x) { acc[n() % KT] = mma<T>(x, frag[n() / KT], acc[n() % KT]); });
  }
  // the same of two tiles with an operand each; a1 comes with its initial values
  template <int KT>
  TURTLE_DEV static void times2(const char* t0, const char* t1, const uint4 (&f0)[STEPS], const uint4 (&f1)[STEPS], f32x16 (&a0)[KT],
                                f32x16 (&a1)[KT], int lane) {
    const uint32_t b0 = row_base(t0, lane), b1 = row_base(t1, lane);
#pragma unroll
    for (int j = 0; j < KT; ++j) a0[j] = zero16();
    in_steps<2 * KT * STEPS, 2>([&](auto n) { return chunk<n() / (2 * KT), n() / 2 % KT>(n() & 1 ? b1 : b0); },
                                     [&](auto n, uint4 x) {
                                       f32x16& a = n() & 1 ? a1[n() / 2 % KT] : a0[n() / 2 % KT];
                                       a = mma<T>(x, n() & 1 ? f1[n() / (2 * KT)] : f0[n() / (2 * KT)], a);
                                     });
  }
  // ... one row group; the second operand read from LDS, from its 32 rows at l1
  TURTLE_DEV static void times2_lds(const char* t0, const char* t1, const uint4 (&f0)[STEPS], const char* l1, f32x16& a0, f32x16& a1,
                                    int lane) {
    const uint32_t b0 = row_base(t0, lane), b1 = row_base(t1, lane);
    uint32_t bl = row_base(l1, lane);
    asm volatile("" : "+v"(bl));      // one address, not a register for each of its chunks
    a0 = zero16();
    uint4 g;
    in_steps<3 * STEPS, 3>([&](auto n) { return chunk<n() / 3, 0>(n() % 3 == 0 ? b0 : n() % 3 == 1 ? bl : b1); },
                           [&](auto n, uint4 x) {
                             if constexpr (n() % 3 == 0) a0 = mma<T>(x, f0[n() / 3], a0);
                             else if constexpr (n() % 3 == 1) g = x;
                             else a1 = mma<T>(x, g, a1);
                           });
  }
  // acc[dt] += (rows 16 U .. 16 U + 15)^T (channels 32 dt ..) x p: 16-bit types, p packed from 8 accumulator registers'
  // values of those rows. LO: a second term of p besides
  template <int U, bool LO>
  TURTLE_DEV static void t_times(const char* t, uint4 hi, uint4 lo, f32x16 (&acc)[DT], int lane) {
    const uint32_t base = tr_base(t, lane);
    static_for<DT>([&](auto dt) {
      const uint32_t a = base ^ (dt() << 6);
      const uint2 x = lds_ld_tr(a + U * 16 * ROWB), y = lds_ld_tr((a ^ 32) + (U * 16 + 8) * ROWB);
      const uint4 v = make_uint4(x.x, x.y, y.x, y.y);
      acc[dt()] = mma<T>(v, hi, acc[dt()]);
      if constexpr (LO) acc[dt()] = mma<T>(v, lo, acc[dt()]);
    });
  }
  // the same for fp32, from register values: row 8 (e >> 2) + (e & 3) + 4 h, channel 32 dt + (lane & 31)
  template <int U>
  TURTLE_DEV static void t_times(const char* t, const float (&p)[8], f32x16 (&acc)[DT], int lane) {
    const int h = lane >> 5;
    static_for<8>([&](auto e) {
      const int row = U * 16 + acc_row(e()) + 4 * h;
      const uint32_t a = lds_addr(t) + row * ROWB + ((((lane & 31) >> 2) ^ swz(row)) << 4) + (lane & 3) * 4;
      static_for<DT>([&](auto dt) {
        acc[dt()] = __builtin_amdgcn_mfma_f32_32x32x2f32(lds_ld4(a ^ (dt() << 7)), p[e()], acc[dt()], 0, 0, 0);
      });
    });
  }
  // V^T operand of rows 16 U .. 16 U + 15, channels 32 dt .. (16-bit types)
  template <int U, int I> TURTLE_DEV static uint4 tr_frag(uint32_t base) {
    const uint32_t a = base ^ (I << 6);
    const uint2 x = lds_ld_tr(a + U * 16 * ROWB), y = lds_ld_tr((a ^ 32) + (U * 16 + 8) * ROWB);
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  // acc += (the tile's 32 KT rows)^T x p, p rounded (16-bit) or as it is (fp32)
  template <int KT>
  TURTLE_DEV static void t_times_all(const char* t, const f32x16 (&p)[KT], f32x16 (&acc)[DT], int lane) {
    if constexpr (ES == 2) {
      uint4 hi[2 * KT];
#pragma unroll
      for (int u = 0; u < 2 * KT; ++u) hi[u] = pack_of(p[u >> 1], 8 * (u & 1));
      const uint32_t base = tr_base(t, lane);
      in_steps<2 * KT * DT, 2>([&](auto n) { return tr_frag<n() / DT, n() % DT>(base); },
                               [&](auto n, uint4 v) { acc[n() % DT] = mma<T>(v, hi[n() / DT], acc[n() % DT]); });
    } else {
      static_for<2 * KT>([&](auto u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[u() >> 1][8 * (u() & 1) + e];
        t_times<u()>(t, x, acc, lane);
      });
    }
  }
  TURTLE_DEV static uint4 pack_of(const f32x16& p, int at) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[at + e];
    return pack(x);
  }
  // sum of the 8 packed values, added to l
  TURTLE_DEV static float sum_packed(uint4 p, float l) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, bf16>::value)
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_, w[i]), bf16x2_{(bf16)1.f, (bf16)1.f}, l, false);
      else if constexpr (ES == 2)
        l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_, w[i]), f16x2_{(f16)1.f, (f16)1.f}, l, false);
    }
    return l;
  }
  TURTLE_DEV static uint4 rest(const float (&p)[8], uint4 hi) {
    typedef T tx8 __attribute__((ext_vector_type(8)));
    const tx8 h = __builtin_bit_cast(tx8, hi);
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = p[i] - (float)h[i];
    return pack(r);
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
  // DMA of N rows of two tensors (LDS tiles t0, t1) by NT threads: src(r, p0, p1) sets the addresses of row r's first
  // channels, or null. For the odd tile: kept small rather than unrolled
  template <int N, int NT, typename F>
  TURTLE_DEV static void load2(char* t0, char* t1, int tid, int D, F src) {
    static_assert(N * CH % NT == 0, "whole DMA instructions");
    const uint32_t b0 = lds_addr(t0) + (uint32_t)(tid & ~63) * 16, b1 = lds_addr(t1) + (uint32_t)(tid & ~63) * 16;
#pragma unroll 1
    for (int i = 0; i < N * CH / NT; ++i) {
      const int ci = i * NT + tid, r = ci / CH, c = ((ci % CH) ^ swz(r)) * 16;
      const char *p0 = nullptr, *p1 = nullptr;
      if (c < D * ES) src(r, p0, p1);
      dma16(p0 ? (const void*)(p0 + c) : (const void*)g_zero_ta, __builtin_amdgcn_readfirstlane(b0 + (uint32_t)i * NT * 16));
      dma16(p1 ? (const void*)(p1 + c) : (const void*)g_zero_ta, __builtin_amdgcn_readfirstlane(b1 + (uint32_t)i * NT * 16));
    }
  }
  // The same where every row is there, row r starts at row 0's address + r st bytes and D = DP. A lane's chunk within
  // its rows depends on the instruction only through the exchange, with a period of NV instructions: its NV offsets
  // are computed once, a tile costs one base address.
  template <int NT> struct Lin {
    static constexpr int RPI = NT / CH, NV = RPI >= 16 ? 1 : 16 / RPI;
    int64_t off[NV];
    TURTLE_DEV void init(int tid, int64_t st) {
#pragma unroll
      for (int i = 0; i < NV; ++i) off[i] = (int64_t)(tid / CH) * st + (((tid % CH) ^ swz(i * RPI + tid / CH)) << 4);
    }
    template <int N>
    TURTLE_DEV void load(char* t, int tid, const char* p, int64_t st) const {
      const uint32_t b0 = lds_addr(t) + (uint32_t)(tid & ~63) * 16;
#pragma unroll
      for (int i = 0; i < N * CH / NT; ++i)
        dma16(p + i * RPI * st + off[i % NV], __builtin_amdgcn_readfirstlane(b0 + (uint32_t)i * NT * 16));
    }
  };
  template <int N, int NT> static constexpr int loads2() { return 2 * (N * CH / NT); }
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
  uint32_t pmul, psh, gmul, gsh;          // j / page = mulhi(j, pmul) >> psh (page > 1); m / G likewise
  const int *table, *kv_lens, *q_lens;
  void *o, *olo;
  float* lse;
  int mtiles, nsplit, total, runs, lds_win;
  float *part, *plse;                     // [nsplit][B Hk][M][D], [nsplit][B Hk][M]
  // backward
  const void* dout;
  int64_t gb, gs, gh;
  void *dq, *dk, *dv;
  const float* delta;
};

// work item of a block. Blocks are dealt to the 8 XCDs in turn, each with an L2 of its own: with enough key heads, runs
// of consecutive items go to one XCD (runs = 1), so that the tiles of a key head share its L2; with few, items are dealt as
// they come (0) - a run would be a piece of one sequence, and pieces cost unequally (causal, documents). Causal items
// of a few rounds of blocks go out longest first over all of an XCD's key heads (2): 5120 tokens, prefix 2048, 16
// heads of 64 channels, dk and dv 210 us for 228, dq 122 for 132, forward 117 for 123.
TURTLE_DEV int xcd_item(const Args& a) {
  if (!a.runs) return (int)blockIdx.x;
  const int x = (int)(blockIdx.x & 7), j = (int)(blockIdx.x >> 3);
  if (a.runs == 2) {
    const int heads = a.B * a.Hk >> 3, n = a.total / (a.B * a.Hk);
    return (x * heads + j % heads) * n + j / heads;
  }
  return x * ((a.total + 7) >> 3) + j;
}

TURTLE_DEV int quot(int n, int d, uint32_t mul, uint32_t sh) { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> sh); }
// the token of row m
TURTLE_DEV int token_of(const Args& a, int m) { return quot(m, a.G, a.gmul, a.gsh); }

// One row's (query's) place and rules, in the lane that owns it
struct Row {
  int pos;       // its place among the keys
  int doc;
  float slope2;
  bool on;
};

TURTLE_DEV Row row_of(const Args& a, int b, int hk, int m, int off, int nq) {
  Row r;
  const int i = token_of(a, m), g = m - i * a.G;
  r.on = m < a.M && i < nq;
  r.pos = i + off;
  r.doc = (a.qdoc && r.on) ? a.qdoc[(int64_t)b * a.Sq + i] : 0;
  if (r.doc < 0) r.on = false;
  r.slope2 = (a.slopes && r.on) ? a.slopes[hk * a.G + g] * LOG2E : 0.f;
  return r;
}

// A row's softmax sum (log2) as the backward takes it, where p = 2^(s - sum): infinity for a row that sees nothing, so all
// its p are 0; where the sum is not a number the least value, so the p of keys it sees are infinite or not a number as
// all that depends on them has to be, and those of hidden ones (s = -infinity) still 0.
TURTLE_DEV float kept_sum(float lse) { return lse == lse ? lse : -3.402823466e38f; }

// tanh of the scores in place, for the cap. While every |x| of the wave is at most 1/2 - scores within half the cap -
// an odd polynomial (least-maximum fit of tanh(x) / x in x^2: relative error 5.5e-7 for 16-bit inputs, 3.3e-9 for
// fp32, to which fp32 arithmetic adds 9e-8): 5 instructions where the exponential form takes two of the slow ones besides.
// Beyond: 16-bit inputs 1 - 2 / (e^2x + 1), off by 1e-7: of a cap up to 64 that is 2^-17, nothing to a 16-bit p; over
// it the wave's values up to 1/2 keep the polynomial (for every cap that would cost 16 % of packed documents at cap 2,
// 25 % of a paged chunk). fp32 the library's.
template <typename T>
TURTLE_DEV float tanh_small(float x) {
  const float u = x * x;
  if constexpr (sizeof(T) == 2) return x * fmaf(u, fmaf(u, fmaf(u, -0.0444022265f, 0.131902966f), -0.333263179f), 0.999999456f);
  else return x * fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -0.0066134277f, 0.0212747076f), -0.0538934189f), 0.13332902f), -0.333333242f), 1.f);
}
template <typename T, int N>
TURTLE_DEV void tanh_all(f32x16 (&s)[N], float icap, float cap) {
  float big = 0.f;
#pragma unroll
  for (int w = 0; w < N; ++w)
#pragma unroll
    for (int r = 0; r < 16; ++r) { s[w][r] *= icap; big = fmaxf(big, fabsf(s[w][r])); }
  auto all = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < N; ++w)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[w][r] = f(s[w][r]);
  };
  if (!__any(!(big <= 0.5f))) {
    all([](float x) { return tanh_small<T>(x); });
  } else if constexpr (sizeof(T) == 4) {
    all([](float x) { return tanhf(x); });
  } else {
    auto far = [](float x) { return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * LOG2E * x)); };
    if (cap <= 64.f) all(far);
    else all([&](float x) { return fabsf(x) <= 0.5f ? tanh_small<T>(x) : far(x); });
  }
}

// document range of tokens [t0, t1): {lo, hi, 1 if all are the same valid number, 1 if any is invalid (backward: or any
// query sees nothing)}
TURTLE_DEV int4 doc_range(const int4* ranges, int nr, int t0, int t1) {
  int4 x = make_int4(0x7fffffff, -1, 1, 0);
  for (int r = t0 / RT; r <= (t1 - 1) / RT && r < nr; ++r) {
    const int4 y = ranges[r];
    x.x = min(x.x, y.x); x.y = max(x.y, y.y); x.z &= y.z; x.w |= y.w;
  }
  if (x.x != x.y) x.z = 0;
  return x;
}

// A walk over tiles of UNIT tokens that may hold a document of [lo, hi]: 64 tiles are looked up at a time, a lane each.
// Of the tile it stops at: mixed = not every pair of it with a pure tile of document `pure` (-1: none) is visible;
// holes = it has tokens without a document; mine = it may hold one of this wave's own documents (own_docs): a block over
// the border of documents walks over all of theirs (forward, 8192 tokens in 7 of 1170, 16 heads on 4, 128 channels: 196 us
// with the waves keeping to their own, 208 without; dk and dv 468 and 464, so there they do not).
struct DocWalk {
  const int4* ranges;     // of this sequence; null: every tile, all visible
  int nr, lo, hi, pure, wlo, whi;
  uint64_t act, mix, hole, own;
  int base;
  bool mixed, holes, mine;
  TURTLE_DEV void none() { ranges = nullptr; nr = 0; lo = hi = pure = wlo = whi = 0; base = -1; act = mix = hole = own = 0; mixed = holes = false; mine = true; }
  // block: the range of the block's tokens
  TURTLE_DEV void init(const int4* r, int n, int4 block) {
    none();
    ranges = r; nr = n; lo = wlo = block.x; hi = whi = block.y; pure = block.z ? block.x : -1;
  }
  // doc: the document of this lane's token, or negative
  TURTLE_DEV void own_docs(int doc) {
    wlo = doc < 0 ? 0x7fffffff : doc; whi = doc;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { wlo = min(wlo, __shfl_xor(wlo, o, 64)); whi = max(whi, __shfl_xor(whi, o, 64)); }
  }
  // the first tile >= t (in steps of `stride`), or `end`; G rows share a token, there are ntok tokens
  template <int UNIT>
  TURTLE_DEV int next(int t, int end, int stride, int G, int ntok, int lane) {
    if (!ranges) return min(t, end);
    while (t < end) {
      if (base < 0 || t >= base + 64 * stride) {
        base = t;
        const int tt = t + lane * stride;
        int4 x = make_int4(0x7fffffff, -1, 0, 0);
        if (tt < end) x = doc_range(ranges, nr, tt * UNIT / G, min((tt * UNIT + UNIT - 1) / G + 1, ntok));
        act = __ballot(x.x <= hi && x.y >= lo);
        mix = __ballot(!(x.z && x.x == pure));
        hole = __ballot(x.w != 0);
        own = __ballot(x.x <= whi && x.y >= wlo);
      }
      const int at = (t - base) / stride;
      const uint64_t left = act >> at;
      if (left) {
        const int k = at + __builtin_ctzll(left);
        mixed = (mix >> k) & 1;
        holes = (hole >> k) & 1;
        mine = (own >> k) & 1;
        return base + k * stride;
      }
      t = base + 64 * stride;
    }
    return end;
  }
};

__device__ const int g_no_doc = -1;

// documents of a tile's N keys -> 256 bytes of LDS, by every wave before the tile's own copy: a register load would be
// waited for in order, behind the tiles in flight. (Waits count the tile's own operations, so with this one more in
// flight they wait for it too: never for less.)
template <int N>
TURTLE_DEV void key_docs(const Args& a, int b, int k0, char* dst, int lane) {
  const int key = k0 + (lane & (N - 1));
  dma4(key < a.Sk ? a.kdoc + (int64_t)b * a.Sk + key : &g_no_doc, __builtin_amdgcn_readfirstlane(lds_addr(dst)));
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

// n / d for n < 2^30: with l = ceil(log2 d), floor(n m / 2^(31 + l)) for m = floor(2^(31 + l) / d) + 1 is exact
void reciprocal(int d, uint32_t& mul, uint32_t& sh) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  mul = d > 1 ? (uint32_t)((1ull << (31 + l)) / (uint64_t)d + 1) : 0;
  sh = d > 1 ? (uint32_t)(l - 1) : 0;
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
  if (!std::isfinite(a.scale2) || !(x->softcap >= 0.f) || !std::isfinite(a.icap) || !std::isfinite(a.cap2)) return false;
  a.slopes = x->slopes; a.prefix = x->prefix; a.qdoc = x->qdoc; a.kdoc = x->kdoc; a.causal = x->causal;
  a.nqr = (x->Sq + RT - 1) / RT; a.nkr = x->table ? 0 : (x->Sk + RT - 1) / RT;
  a.qr = (const int4*)x->ranges; a.kr = a.qr ? a.qr + (int64_t)x->B * a.nqr : nullptr;
  a.page = x->page; a.npages = x->npages; a.maxpages = x->maxpages; a.table = x->table; a.kv_lens = x->kv_lens; a.q_lens = x->q_lens;
  if (x->table) reciprocal(x->page, a.pmul, a.psh);
  reciprocal(a.G, a.gmul, a.gsh);
  a.o = x->o; a.olo = dtype == 0 ? nullptr : x->o_lo; a.lse = x->lse;
  return true;
}

template <typename K>
int launch(K kernel, int64_t total, int threads, int lds, Args& a, hipStream_t st) {
  if (total <= 0 || total >= (1ll << 30)) return -1;
  const int bh = a.B * a.Hk;
  a.total = (int)total;
  a.runs = bh % 8 == 0 || bh >= 64;
  if (a.causal && bh % 8 == 0 && total <= 8 * 256) a.runs = 2;
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return (int)e;
  }
  kernel<<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(threads), lds, st>>>(a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace turtle
