// What the attention kernels over a cache share, of bf16 rows (attention.hip) and of
// 8-bit codes (attention8.hip): how key tiles are dealt over workgroups, a wave's rows
// with their running softmax, and the joins of what several workgroups computed.
#pragma once

#include <algorithm>

#include "common.hpp"
#include "gemm_ks.hpp"  // device_cus

namespace umic {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kStep = 32;             // keys of a wave's step

struct AttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  const int32_t* table;   // or NULL: request b is block b
  const int32_t* kv_len;  // or NULL: len
  const int32_t* q_len;   // or NULL: S
  int32_t* counters;      // [nwg], zero between calls; NULL: a second kernel joins the parts
  float* part;            // [2 nwg][rows of a block][D]
  float* part_ml;         // [2 nwg][rows of a block] (max, sum)
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss, c_sb, c_sh, table_ld;
  int cap;                // keys a request can hold
  int c_ss;               // below 2^24: row offsets inside a tile are 32-bit
  int B, S, Hk, G, rb;    // rb: row blocks of a (request, key head)
  int len, blocks, shift, causal, nwg, some;  // nwg, some: see Deal
  uint32_t flip;          // sign bits of q (a negative scale)
  float c;                // |scale| * log2(e)
};

// The kernel's arguments, loaded again: held over the loops, they and what follows from
// them do not fit the scalar registers.
__device__ __forceinline__ AttnArgs args_again() {
  typedef const __attribute__((address_space(4))) AttnArgs* Args;
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttnArgs*)p;
}

// A scalar load whatever the compiler can prove about the kernel's stores.
__device__ __forceinline__ int scalar_i32(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

// x / y of numbers that are not negative: fewer instructions than signed ones take.
__device__ __forceinline__ int quot(int x, int y) { return (int)((unsigned)x / (unsigned)y); }

__device__ __forceinline__ int len_of(const AttnArgs& a, int b) {
  return a.kv_len ? min(max(scalar_i32(a.kv_len + b), 0), a.cap) : a.len;
}

__device__ __forceinline__ int new_of(const AttnArgs& a, int b) {
  return a.q_len ? min(max(scalar_i32(a.q_len + b), 0), a.S) : a.S;
}

// How a launch's key tiles are dealt.  A segment is one (request, key head, row
// block); it counts as its tiles and LEAD more, what its start and end cost.  The
// first `more` workgroups have each + 1 of the sum, the others each.
template <int TILE, int LEAD, int LEAST, int EACH = LEAST>
struct Deal {
  unsigned each, more;
  int nwg;

  static __device__ __forceinline__ int tiles(int keys) { return (keys + TILE - 1) / TILE; }
  static __device__ __forceinline__ int units(int keys) {
    return keys > 0 ? tiles(keys) + LEAD : 0;
  }
  // most: that the chip holds; if that many have no work (LEAST units each), no more than
  // `some`, of EACH or more
  __device__ __forceinline__ Deal(unsigned all, int most, int some) {
    const unsigned fit = (all + LEAST - 1) / LEAST;
    nwg = fit >= (unsigned)most ? most : min((int)((all + EACH - 1) / EACH), some);
    each = nwg ? all / (unsigned)nwg : 0;
    more = all - each * (unsigned)nwg;
  }
  __device__ __forceinline__ int begin(unsigned wg) const {
    return (int)(wg * each + (wg < more ? wg : more));
  }
  __device__ __forceinline__ int holder(unsigned unit) const {
    const unsigned wide = more * (each + 1);
    return (int)(unit < wide ? unit / (each + 1) : more + (unit - wide) / each);
  }
  // the workgroups that hold a segment's first and last tile; it begins at unit `at`
  __device__ __forceinline__ void holders(unsigned at, int tiles, int& w0, int& w1) const {
    w0 = holder(at + LEAD);
    w1 = holder(at + LEAD + tiles - 1);
  }
};
typedef Deal<kStep * kWaves, 0, 1> FewDeal;  // single tokens: 128 keys, as they are
// Many rows: a segment's start and end cost some four steps of 32 keys.  (LEAD, LEAST)
// = (4, 4): 32 tokens over 256 keys 12.9 us, over 3126 18.8, four 128-token chunks 51;
// (2, 3): 12.3, 21.4, 57; (4, 3): 12, 21, 51; (4, 8): 18.9, 20.2, 51.
typedef Deal<kStep, 4, 4> ManyDeal;

// Units of all requests, and those before this thread's requests (a contiguous
// share of them: [first, end)).
struct Scan {
  int all, before, first, end;
};

template <typename DEAL>
__device__ __forceinline__ Scan scan_units(const AttnArgs& a, int* sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int share = (a.B + kThreads - 1) / kThreads;
  Scan s;
  s.first = min(a.B, (int)threadIdx.x * share);
  s.end = min(a.B, s.first + share);
  int n = 0;
  for (int i = s.first; i < s.end; ++i) n += DEAL::units(min(max(a.kv_len[i], 0), a.cap));
  int x = n;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  if (lane == kWave - 1) sums[wave] = x;
  __syncthreads();
  s.all = 0;
  s.before = x - n;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    s.all += sums[w];
    if (w < wave) s.before += sums[w];
  }
  return s;
}

// Part of a segment: its place in the launch, tiles [t0, t1).
struct Segment {
  int b, h, rb, len, tiles, t0, t1, fresh, at;
};

// A workgroup's walk over its segments.  BLOCKS: a (request, key head) can have more
// than one row block.
template <typename DEAL, bool BLOCKS>
struct Walk {
  int u, u_end, b, before, per;

  __device__ __forceinline__ void start(const AttnArgs& a, const DEAL& deal, const Scan& scan,
                                        int even, int wg, int* found) {
    per = BLOCKS ? a.Hk * a.rb : a.Hk;
    u = deal.begin(wg);
    u_end = deal.begin(wg + 1);
    const int target = quot(u, per);
    if (a.kv_len) {
      int x = scan.before;
      for (int i = scan.first; i < scan.end; ++i) {
        const int n = DEAL::units(min(max(a.kv_len[i], 0), a.cap));
        if (target >= x && target < x + n) {
          found[0] = i;
          found[1] = x;
        }
        x += n;
      }
      __syncthreads();
      b = __builtin_amdgcn_readfirstlane(found[0]);
      before = __builtin_amdgcn_readfirstlane(found[1]);
    } else {
      b = quot(target, even);
      before = b * even;
    }
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, Segment& s) {
    while (u < u_end) {
      s.len = len_of(a, b);
      const int units = DEAL::units(s.len);
      if (units == 0) {
        ++b;
        continue;
      }
      s.tiles = DEAL::tiles(s.len);
      const int lead = units - s.tiles;
      const int in = u - before * per;
      const int pair = quot(in, units);
      const int p0 = in - pair * units, p1 = min(units, p0 + u_end - u);
      s.at = before * per + pair * units;
      s.b = b;
      s.h = BLOCKS ? quot(pair, a.rb) : pair;
      s.rb = BLOCKS ? pair - s.h * a.rb : 0;
      s.t0 = max(0, p0 - lead);
      s.t1 = max(0, p1 - lead);
      s.fresh = new_of(a, b);
      u += p1 - p0;
      if (u - before * per >= units * per) {
        before += units;
        ++b;
      }
      if (s.t1 > s.t0) return true;
    }
    return false;
  }
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ bf16x8_t as_bf(const u32x4& v) {
  return __builtin_bit_cast(bf16x8_t, v);
}

// The low (hi: high) halves of two words side by side.
__device__ __forceinline__ uint32_t pair_lo(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t pair_hi(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// A segment's keys: row j is row j % 2^shift of block row[j >> shift], and base is
// row 0 of block 0; row NULL: all are one block.
struct Keys {
  int64_t base;
  const int32_t* row;
  int len;
};

__device__ __forceinline__ Keys keys_of(const AttnArgs& a, const Segment& s) {
  Keys k;
  k.row = a.table ? a.table + s.b * a.table_ld : nullptr;
  k.base = s.h * a.c_sh + (a.table ? 0 : s.b * a.c_sb);
  k.len = s.len;
  return k;
}

// The blocks of 32 keys from k0 on: of two tiles of 16 (a block never ends inside
// one).  Asked for a step before their place is needed.
struct Blocks {
  int of[2];
};

__device__ __forceinline__ Blocks blocks_of(const AttnArgs& a, const Keys& s, int k0) {
  Blocks x = {};
  if (s.row) {
    const int last = (s.len - 1) >> a.shift;
    x.of[0] = scalar_i32(s.row + min(k0 >> a.shift, last));
    x.of[1] = scalar_i32(s.row + min((k0 + 16) >> a.shift, last));
  }
  return x;
}

// Where the two tiles lie, the first `n` rows of each there.
struct Place {
  int64_t at[2];
  int n[2];
};

__device__ __forceinline__ Place place_of(const AttnArgs& a, const Keys& s, int k0,
                                          const Blocks& x) {
  Place p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int key = k0 + 16 * i;
    p.n[i] = min(max(s.len - key, 0), 16);
    // a block outside the pool: not there; rows that are not there are read elsewhere
    const unsigned block = (unsigned)x.of[i];
    if (block >= (unsigned)a.blocks) p.n[i] = 0;
    p.at[i] = s.base;
    if (p.n[i]) p.at[i] += block * a.c_sb + (int64_t)(key & ((1 << a.shift) - 1)) * a.c_ss;
  }
  return p;
}

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < __builtin_inff(); }

// Values that are not finite.  Every key a row sees has a weight above 0, so an
// infinite v makes its column infinite, and two of both signs, or a NaN, make it NaN.
// The products do not give that: the weight's low part is negative or 0, and 0 and
// what underflows times infinity is NaN.  But whatever they give is not finite, and
// stays so: where a row's o (of N groups of four columns, col + STEP g ..) is not, the
// values among keys [from, to) below lim that are not finite take its place.  (Sums of
// finite values that overflowed have none, and stay.)  count: of rows that are written,
// and not NaN as their weights are.
template <int N, int STEP>
__device__ __forceinline__ void restore(f32x4_t (&o)[N], bool count, const AttnArgs& a, const Keys& s,
                                        int from, int to, int lim, int col) {
  float none = 0.0f;  // NaN: not all are finite
#pragma unroll
  for (int g = 0; g < N; ++g)
#pragma unroll
    for (int y = 0; y < 4; ++y) none = __builtin_fmaf(o[g][y], 0.0f, none);
  if (!__any(count && none != none)) return;
  f32x4_t sum[N] = {};
#pragma unroll 1
  for (int k0 = from; k0 < to; k0 += kStep) {
    const Place p = place_of(a, s, k0, blocks_of(a, s, k0));
#pragma unroll 1
    for (int key = 0; key < kStep; ++key) {
      const int at = key & 15;
      if (at >= (key < 16 ? p.n[0] : p.n[1])) continue;
      const uint16_t* vp = a.v + (key < 16 ? p.at[0] : p.at[1]) + (int64_t)at * a.c_ss + col;
      u32x2 raw[N];
#pragma unroll
      for (int g = 0; g < N; ++g) raw[g] = *reinterpret_cast<const u32x2*>(vp + STEP * g);
#pragma unroll
      for (int g = 0; g < N; ++g) {
        float x[4];
        unpack4(raw[g], x);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (k0 + key < lim && !finite(x[y])) sum[g][y] += x[y];
      }
    }
  }
#pragma unroll
  for (int g = 0; g < N; ++g)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (sum[g][y] != 0.0f) o[g][y] = sum[g][y];
}

// A wave's rows r0 .. of a segment (row r is head r % G of new token r / G), NT
// tiles of 16, a lane's being n16 of each; and what a step of 32 keys does to
// them.  The V operand of output tile e holds for a lane one column of 8 keys, j =
// 4 i + y being key 16 i + 4 g4 + y.  TURNED: it comes so from LDS, v[4 e ..] its
// words, column 16 e + n16.  Else v[VW j ..] are DV columns of key j from DV n16 on,
// turned in registers, tile e being column DV n16 + e of each lane.
template <int D, int NT, bool TURNED>
struct Rows {
  static constexpr int KK = D / 32;  // 32-wide steps of a score's product
  static constexpr int DV = D / 16;  // output columns of a lane, V columns it reads
  static constexpr int VW = DV / 2;  // 32-bit words of those
  static constexpr int VR = 8 * VW;  // words of V a lane holds
  static constexpr float kSlack = 8.0f;
  u32x4 q[NT][KK];
  int lim[NT];  // keys below it are seen
  int lo, hi;   // keys below lo are seen by all rows, keys from hi on by none
  // p is exp2(c (score - base)); base is 0 until a key is seen, and what reaches top is
  // followed
  float base[NT], top[NT], l[NT];
  f32x4_t acc[NT][DV];

  __device__ __forceinline__ float max_of(int nt) const {
    return top[nt] == -__builtin_inff() ? top[nt] : base[nt];
  }

  // WIDE: a lane's operand of two steps is 16 neighbouring elements of the key.
  template <bool WIDE = false>
  __device__ __forceinline__ void load_q(const AttnArgs& a, const Segment& s, int r0, int n16,
                                         int g4) {
    const int rows = a.S * a.G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = min(r0 + nt * 16 + n16, rows - 1);  // past them: computed, not written
      const int t = quot(r, a.G), g = r - t * a.G;
      lim[nt] = a.causal ? min(s.len, s.len - s.fresh + t + 1) : s.len;
      const uint16_t* qp =
          a.q + s.b * a.q_sb + (int64_t)(s.h * a.G + g) * a.q_sh + t * a.q_ss + g4 * (WIDE ? 16 : 8);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        q[nt][kk] = *reinterpret_cast<const u32x4*>(
                        qp + (WIDE ? (kk >> 1) * 64 + (kk & 1) * 8 : kk * 32)) ^ a.flip;
    }
    lo = hi = s.len;
    if (a.causal) {
      lo = min(s.len, s.len - s.fresh + quot(min(r0, rows - 1), a.G) + 1);
      hi = min(s.len, s.len - s.fresh + quot(min(r0 + 16 * NT, rows) - 1, a.G) + 1);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      base[nt] = l[nt] = 0.0f;
      top[nt] = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < DV; ++e) acc[nt][e] = f32x4_t{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void scores(const u32x4 (&kf)[2][KK], f32x4_t (&sc)[NT][2]) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[nt][i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          sc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(kf[i][kk]), as_bf(q[nt][kk]),
                                                               sc[nt][i], 0, 0, 0);
  }
  // Output column of acc[..][e][y].
  static __device__ __forceinline__ int column(int e, int y, int g4) {
    return TURNED ? 16 * e + 4 * g4 + y : (4 * g4 + y) * DV + e;
  }
  // Keys that are not there, and those a row does not see.
  __device__ __forceinline__ void mask(f32x4_t (&sc)[NT][2], uint32_t (&v)[VR], const int (&n)[2],
                                       int k0, int g4) const {
    uint32_t keep[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = 4 * g4 + (j & 3), key = k0 + 16 * (j >> 2) + at;
      const bool there = at < n[j >> 2];
      keep[j] = there ? 0xffffffffu : 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (!there || key >= lim[nt]) sc[nt][j >> 2][j & 3] = -__builtin_inff();
    }
    // 0 * inf is not 0
#pragma unroll
    for (int x = 0; x < VR; ++x) {
      const int j = TURNED ? (x & 3) * 2 : x / VW;
      v[x] &= TURNED ? (keep[j] & 0xffffu) | (keep[j + 1] & 0xffff0000u) : keep[j];
    }
  }
  // p of the scores, in two bf16 parts.  The base follows a row's maximum only when it
  // is passed by kSlack: p stays below 2^kSlack, and the outputs are rescaled a few
  // times in all.  The base is a score, not a rounded exponent: with fma(score, c, -base)
  // a base above 2^31 leaves its own rounding as the exponent of the maximum.  (One more
  // instruction an element, 1 to 2% of a step: 128 tokens over 65536 keys 226 us for 223.)
  // SCALED: p comes times the scale of its key's v (vs: of the two tiles), its sum without.
  template <bool SCALED = false>
  __device__ __forceinline__ void weights(const f32x4_t (&sc)[NT][2], float c, u32x4 (&ph)[NT],
                                          u32x4 (&pl)[NT], const float* vs = nullptr) {
    float x[NT][8];
    auto most = [&](int nt) {  // of exponents, which need no quieting of NaNs first
      const float(&y)[8] = x[nt];
      return fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])),
                   fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
    };
    auto exponents = [&](int nt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[nt][j] = (sc[nt][j >> 2][j & 3] - base[nt]) * c;
    };
    bool up = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      exponents(nt);
      up |= most(nt) >= top[nt];  // -inf too, ahead of a base: the product with c overflows
    }
    if (__any(up)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float from = max_of(nt);
        float mx = sc[nt][0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, sc[nt][j >> 2][j & 3]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        const float to = fmaxf(from, mx);
        if (to > -__builtin_inff()) {
          const float al = __builtin_amdgcn_exp2f((from - to) * c);
          base[nt] = to;
          top[nt] = kSlack;
          l[nt] *= al;
#pragma unroll
          for (int e = 0; e < DV; ++e) acc[nt][e] *= al;
        }
        exponents(nt);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[nt][j] = __builtin_amdgcn_exp2f(x[nt][j]);
        l[nt] += x[nt][j];
        if constexpr (SCALED) x[nt][j] *= vs[j >> 2];
      }
      ph[nt] = pack8(x[nt]);
      unpack8(ph[nt], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[nt][j] - y[j];
      pl[nt] = pack8(y);
    }
  }
  // Where some rows do not see some of the keys, p = 0 has to hide a v that is not
  // finite, and 0 * inf is not 0: such elements leave the product, and the rows that
  // see them are marked by them, for `restore`.
  __device__ __forceinline__ void hide(uint32_t (&v)[VR], const AttnArgs& a, const Place& p, int k0,
                                       int g4) {
    // exponents of ones, both halves of a word at once: bits 15 and 31
    auto wild = [](uint32_t x) { return (x & 0x7f807f80u) + 0x00800080u; };
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < VR; ++w) any |= wild(v[w]);
    if (!__any(any & 0x80008000u)) return;
#pragma unroll
    for (int w = 0; w < VR; ++w) v[w] &= ~((wild(v[w]) >> 15 & 0x00010001u) * 0xffffu);
#pragma unroll 1
    for (int key = 0; key < kStep; ++key) {
      const int at = key & 15;
      if (at >= (key < 16 ? p.n[0] : p.n[1])) continue;
      const uint16_t* vp = a.v + (key < 16 ? p.at[0] : p.at[1]) + (int64_t)at * a.c_ss;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (k0 + key < lim[nt])
#pragma unroll
          for (int e = 0; e < DV; ++e)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float x = bf2f(vp[column(e, y, g4)]);
              if (!finite(x)) acc[nt][e][y] += x;
            }
    }
  }
  __device__ __forceinline__ void product(const uint32_t (&v)[VR], const u32x4 (&ph)[NT],
                                          const u32x4 (&pl)[NT]) {
#pragma unroll
    for (int w = 0; w < VW; ++w) {  // two tiles at a time
      u32x4 v0, v1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TURNED) {
          v0[j] = v[8 * w + j];
          v1[j] = v[8 * w + 4 + j];
        } else {
          v0[j] = pair_lo(v[2 * j * VW + w], v[(2 * j + 1) * VW + w]);
          v1[j] = pair_hi(v[2 * j * VW + w], v[(2 * j + 1) * VW + w]);
        }
      }
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bf16x8_t p = as_bf(part ? pl[nt] : ph[nt]);
          f32x4_t& c0 = acc[nt][2 * w];
          f32x4_t& c1 = acc[nt][2 * w + 1];
          c0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v0), p, c0, 0, 0, 0);
          c1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v1), p, c1, 0, 0, 0);
        }
    }
  }
};

// Stores and loads that other XCDs' workgroups see and are seen by: agent-scope
// accesses, which pass the XCD's own cache by.  (With plain ones between
// __threadfence() calls every workgroup wrote its XCD's cache back and emptied it:
// 64 ragged requests took three times as long as with a second kernel.)
__device__ __forceinline__ void put2(float* p, float x, float y) {
  const uint64_t v = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint16_t* out_row(const AttnArgs& a, int b, int h, int r) {
  const int t = quot(r, a.G), g = r - t * a.G;
  return a.out + b * a.o_sb + t * a.o_ss + (int64_t)(h * a.G + g) * a.o_sh;
}

// One row tile of a wave of many rows, as the lanes hold it: rows of the output, or a part
// in the workspace (slot).  row: the lane's; sum: of its weights.
template <int D, int NT, typename R>
__device__ __forceinline__ void write_rows(const AttnArgs& args, const Segment& seg, const R& r,
                                           int nt, int row, int slot, bool padded, float sum) {
  constexpr int DV = R::DV;
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // a lane's columns: 16 e + 4 g4 .. + 4
  if (seg.t0 == 0 && seg.t1 == seg.tiles) {
    const bool none = padded || sum == 0.0f;
    const float inv = 1.0f / sum;
    uint16_t* op = out_row(args, seg.b, seg.h, row) + 4 * g4;
#pragma unroll
    for (int e = 0; e < DV; ++e) {
      const f32x4_t x = r.acc[nt][e] * inv;
      const u32x2 o = {none ? 0 : pack2(x[0], x[1]), none ? 0 : pack2(x[2], x[3])};
      *reinterpret_cast<u32x2*>(op + 16 * e) = o;
    }
  } else {
    // as the lanes hold them, side by side: the join reads them the same way
    const int64_t tile = (int64_t)slot * (NT * kWaves) + wave * NT + nt;
    f32x4_t* p = reinterpret_cast<f32x4_t*>(args.part) + tile * 4 * D + lane;
#pragma unroll
    for (int e = 0; e < DV; ++e) p[e * kWave] = r.acc[nt][e];
    if (g4 == 0) {
      args.part_ml[(tile * 16 + n16) * 2] = r.max_of(nt);
      args.part_ml[(tile * 16 + n16) * 2 + 1] = sum;
    }
  }
}

// Joins one row of a segment that workgroups w0 .. w1 hold, a wave to a row.  Part i,
// 64 of them at a time: lane i holds its maximum and sum, D / 4 lanes a fourth of its
// columns each.  The first part is its workgroup's second (its last segment), the
// others their first; loads past the last give zeros.  SHARED: the parts were written
// by this launch.  (With 32 parts in flight, each by its own address, the code was
// three times as long, and fetching it what the join waited for: a single token over
// 3100 keys, 25 parts, 12.4 us for 10.4.)
template <int D, bool SHARED>
__device__ __forceinline__ void join_row(const AttnArgs& a, int w0, int w1, int rr, bool none,
                                         uint16_t* op) {
  constexpr int kLanes = D / 4, kParts = kWave / kLanes;  // lanes of a part, parts a load
  constexpr int kAhead = 8;
  constexpr int kAux = SHARED ? 16 : 0;  // sc1: agent scope
  constexpr int kRow = 16 * D * 4, kRowMl = 16 * 2 * 4;   // bytes from a slot to the next
  const int lane = threadIdx.x & (kWave - 1);
  const int sub = lane / kLanes, col = (lane & (kLanes - 1)) * 4;
  const int n = w1 - w0 + 1;  // two at least
  const int64_t first = (int64_t)w0 * 2 * 16 + rr;
  const auto parts = __builtin_amdgcn_make_buffer_rsrc(a.part + first * D, 0, (2 * n - 1) * kRow,
                                                       0x00020000);
  const auto mls = __builtin_amdgcn_make_buffer_rsrc(a.part_ml + first * 2, 0,
                                                     (2 * n - 1) * kRowMl, 0x00020000);
  auto slot_of = [](int i) { return 2 * i + (i == 0); };
  float mi, li;  // part `lane`'s
  auto load_ml = [&](int i) {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(mls, slot_of(i) * kRowMl, 0, kAux);
    mi = i < n ? __uint_as_float(x[0]) : -__builtin_inff();
    li = __uint_as_float(x[1]);
  };
  f32x4_t x[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      x[j] = __builtin_bit_cast(
          f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                       parts, slot_of(i0 + j * kParts + sub) * kRow + col * 4, 0, kAux));
  };
  load_ml(lane);
  load(0);
  float mx = mi;
  for (int i0 = kWave; i0 < n; i0 += kWave) {
    load_ml(i0 + lane);
    mx = fmaxf(mx, mi);
  }
  if (n > kWave) load_ml(lane);
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) mx = fmaxf(mx, __shfl_xor(mx, k, kWave));
  const float base = mx == -__builtin_inff() ? 0.0f : mx;
  f32x4_t o = {0, 0, 0, 0};
  float sum = 0.0f;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kWave) {
    if (i0) load_ml(i0 + lane);
    const float f = __builtin_amdgcn_exp2f((mi - base) * a.c);
    sum += li * f;
#pragma unroll 1
    for (int j0 = 0; j0 < kWave && i0 + j0 < n; j0 += kAhead * kParts) {
      if (i0 + j0) load(i0 + j0);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) o += x[j] * __shfl(f, j0 + j * kParts + sub, kWave);
    }
  }
#pragma unroll
  for (int k = kLanes; k < kWave; k <<= 1)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], k, kWave);
  if (__any(!none && !(finite(o[0]) && finite(o[1]) && finite(o[2]) && finite(o[3])))) {
    f32x4_t whole = {0, 0, 0, 0};  // of the parts that are not finite, whatever their weight
#pragma unroll 1
    for (int i = 0; i < n; i += kAhead * kParts) {
      load(i);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) whole[c] += finite(x[j][c]) ? 0.0f : x[j][c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int k = kLanes; k < kWave; k <<= 1) whole[c] += __shfl_xor(whole[c], k, kWave);
      if (whole[c] != 0.0f) o[c] = whole[c];
    }
  }
  sum = group_sum<kWave>(sum);
  if (sum == 0.0f) none = true;
  const u32x2 out = {none ? 0 : pack2(o[0] / sum, o[1] / sum),
                     none ? 0 : pack2(o[2] / sum, o[3] / sum)};
  if (sub == 0) *reinterpret_cast<u32x2*>(op + col) = out;
}

// Requests without a key: zeros (of up to 16 rows a key head: their count is 32-bit).
template <int D>
__device__ __forceinline__ void zero_rows(const AttnArgs& a) {
  constexpr int chunks = D / 8;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (len_of(a, b)) continue;
    const int heads = a.Hk * a.G;
    for (int i = threadIdx.x; i < a.S * heads * chunks; i += kThreads) {
      const int c = i & (chunks - 1), row = i / chunks;
      const int t = quot(row, heads), h = row - t * heads;
      uint16_t* op = a.out + b * a.o_sb + t * a.o_ss + (int64_t)h * a.o_sh + c * 8;
      *reinterpret_cast<u32x4*>(op) = u32x4{0, 0, 0, 0};
    }
  }
}

// What attend_few's waves share of a workgroup's LDS.
template <int D>
struct alignas(16) FewShared {
  float acc[kWaves][16][D + 4];  // first: read and written 16 bytes at a time
  float ml[kWaves][16][2];
  int sums[kWaves];
  int found[2];
  int arrived[2];
  Segment kept[2];  // those that other workgroups have a part of: the first, the last
};

// Joins the waves of a workgroup that has done a segment's tiles: rows of the output, or a
// part in the workspace.  RESTORE: v can hold values that are not finite.
template <int D, bool RESTORE, typename R>
__device__ __forceinline__ void join_waves(const AttnArgs& args, R& r, const Segment& seg,
                                           FewShared<D>& lds, int wg, int& split) {
  constexpr int DV = R::DV, VW = R::VW;
  constexpr int kTile = kStep * kWaves;
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rows = args.S * args.G;
  const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
  const int slot = wg * 2 + (seg.t0 == 0 ? 1 : 0);
  r.l[0] += __shfl_xor(r.l[0], 16, kWave);
  r.l[0] += __shfl_xor(r.l[0], 32, kWave);
  if (g4 == 0) {
    lds.ml[wave][n16][0] = r.max_of(0);
    lds.ml[wave][n16][1] = r.l[0];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < DV; ++e) lds.acc[wave][n16][(4 * g4 + i) * DV + e] = r.acc[0][e][i];
  __syncthreads();
  // thread: row tid / 16, columns DV (tid % 16) ..
  const int rr = threadIdx.x >> 4, col = (threadIdx.x & 15) * DV;
  if (rr < rows) {
    float mx = lds.ml[0][rr][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, lds.ml[w][rr][0]);
    const float base = mx == -__builtin_inff() ? 0.0f : mx;
    f32x4_t o[DV / 4] = {};
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f((lds.ml[w][rr][0] - base) * args.c);
      sum += lds.ml[w][rr][1] * f;
#pragma unroll
      for (int e = 0; e < DV; ++e) o[e / 4][e % 4] += lds.acc[w][rr][col + e] * f;
    }
    const int token = quot(rr, args.G);
    const int lim = args.causal ? seg.len - seg.fresh + token + 1 : seg.len;
    if constexpr (RESTORE)
      restore<DV / 4, 4>(o, token < seg.fresh && sum == sum, args, keys_of(args, seg),
                       seg.t0 * kTile, seg.t1 * kTile, lim, col);
    if (whole) {
      const bool none = token >= seg.fresh || sum == 0.0f;
      const float inv = 1.0f / sum;
      uint32_t* op = reinterpret_cast<uint32_t*>(out_row(args, seg.b, seg.h, rr) + col);
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const f32x4_t& x = o[w / 2];
        op[w] = none ? 0 : pack2(x[w % 2 * 2] * inv, x[w % 2 * 2 + 1] * inv);
      }
    } else {
      const int64_t at = (int64_t)slot * 16 + rr;
#pragma unroll
      for (int e = 0; e < DV; e += 2)
        put2(args.part + at * D + col + e, o[e / 4][e % 4], o[e / 4][e % 4 + 1]);
      if (col == 0) put2(args.part_ml + at * 2, mx, sum);
    }
  }
  if (!whole) {
    split |= seg.t0 == 0 ? 2 : 1;
    if (threadIdx.x == 0) lds.kept[seg.t0 == 0 ? 1 : 0] = seg;
  }
  __syncthreads();  // LDS is used again
}

// Joins the segments of which this workgroup's parts are the last to come.
template <int D, typename DEAL>
__device__ __forceinline__ void join_parts(const AttnArgs& args, const DEAL& deal,
                                           FewShared<D>& lds, int split) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rows = args.S * args.G;
  if (args.counters && split) {
    // Both parts are counted at the end: a count after each kept the workgroup
    // waiting while none of its loads were on their way.  Every wave's stores have
    // arrived before.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int w0[2], w1[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!(split >> i & 1)) continue;
      deal.holders(uniform(lds.kept[i].at), uniform(lds.kept[i].tiles), w0[i], w1[i]);
      if (threadIdx.x == 0)
        lds.arrived[i] = __hip_atomic_fetch_add(args.counters + w0[i], 1, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const int v0 = i ? w0[1] : w0[0], v1 = i ? w1[1] : w1[0];
      // others' parts are missing
      if (!(split >> i & 1) || uniform(lds.arrived[i]) != v1 - v0) continue;
      if (threadIdx.x == 0) args.counters[v0] = 0;  // for the next call
      const int b = uniform(lds.kept[i].b), h = uniform(lds.kept[i].h), fresh = uniform(lds.kept[i].fresh);
      for (int row = wave; row < rows; row += kWaves)
        join_row<D, true>(args, v0, v1, row, quot(row, args.G) >= fresh,
                          out_row(args, b, h, row));
    }
  }
}

// This workgroup's place in the deal: they go round the eight XCDs, and those of
// one XCD take neighbouring tiles.
__device__ __forceinline__ int dealt_wg(int nwg) {
  const int eighth = (nwg + 7) / 8;
  const int wg = (blockIdx.x & 7) * eighth + blockIdx.x / 8;
  return (int)(blockIdx.x / 8) < eighth && wg < nwg ? wg : -1;
}

// All but LEFT of this wave's loads have landed and its LDS reads are done; then
// the workgroup's barrier.  No memory access moves across.
template <int LEFT>
__device__ __forceinline__ void landed_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | (7 << 4) | ((LEFT >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

// What a join needs to know of its (request, key head, row block).
template <typename DEAL>
__device__ __forceinline__ bool find_parts(const AttnArgs& a, int b, int pair, int* sums,
                                           int* found, int& w0, int& w1) {
  const int per = a.Hk * a.rb;
  const int len = len_of(a, b), tiles = DEAL::tiles(len), units = DEAL::units(len);
  int all = units * a.B, before = units * b;
  if (a.kv_len) {
    const Scan scan = scan_units<DEAL>(a, sums);
    all = scan.all;
    if (b >= scan.first && b < scan.end) {
      int x = scan.before;
      for (int i = scan.first; i < b; ++i) x += DEAL::units(min(max(a.kv_len[i], 0), a.cap));
      *found = x;
    }
    __syncthreads();
    before = *found;
  }
  w0 = 0, w1 = -1;
  if (tiles == 0) return false;
  const DEAL deal((unsigned)(all * per), a.nwg, a.some);
  deal.holders((unsigned)(before * per + pair * units), tiles, w0, w1);
  return true;
}

// Joins the parts that attend_few_kernel has left, and writes the zeros.
template <int D, typename DEAL>
__global__ __launch_bounds__(kThreads) void join_few_kernel(AttnArgs a) {
  __shared__ int sums[kWaves];
  __shared__ int found;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int b = blockIdx.x / a.Hk, h = blockIdx.x - b * a.Hk;
  int w0, w1;
  const bool any = find_parts<DEAL>(a, b, h, sums, &found, w0, w1);
  const int row = blockIdx.y * kWaves + wave;
  if (row >= a.S * a.G) return;
  uint16_t* op = out_row(a, b, h, row);
  if (!any)
    for (int c = threadIdx.x & (kWave - 1); c < D; c += kWave) op[c] = 0;
  else if (w0 != w1)
    join_row<D, false>(a, w0, w1, row, quot(row, a.G) >= new_of(a, b), op);
}

// Joins those of attend_many_kernel: a workgroup to 4 of the DV column groups of a
// tile of 16 rows, a lane to four columns of one row.
template <int D, int NT, typename DEAL>
__global__ __launch_bounds__(kThreads) void join_many_kernel(AttnArgs a) {
  constexpr int DV = D / 16;
  constexpr int kBlock = 16 * NT * kWaves, kTiles = kBlock / 16;
  __shared__ int sums[kWaves];
  __shared__ int found;
  const int lane = threadIdx.x & (kWave - 1), n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int per = a.Hk * a.rb;
  const int b = blockIdx.x / per, pair = blockIdx.x - b * per;
  const int h = pair / a.rb, rb = pair - h * a.rb;
  int w0, w1;
  const bool any = find_parts<DEAL>(a, b, pair, sums, &found, w0, w1);
  const int group = blockIdx.z * kWaves + wave;
  const int row = rb * kBlock + blockIdx.y * 16 + n16;
  if ((any && w0 == w1) || group >= DV || row >= a.S * a.G) return;
  const int n = w1 - w0 + 1;
  const int64_t first = (int64_t)w0 * 2 * kTiles + blockIdx.y;
  auto tile_of = [&](int i) { return first + (2 * i + (i == 0)) * kTiles; };
  const float* ml = a.part_ml + n16 * 2;
  const f32x4_t* part = reinterpret_cast<const f32x4_t*>(a.part) + group * kWave + lane;
  // kAhead parts at a time, all their loads at once
  constexpr int kAhead = 8;
  float mx = -__builtin_inff(), sum = 0.0f;
  f32x4_t o = {0, 0, 0, 0};
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float m[kAhead], l[kAhead];
    f32x4_t x[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t t = tile_of(min(i0 + j, n - 1));
      m[j] = ml[t * 32], l[j] = ml[t * 32 + 1];
      x[j] = part[t * 4 * D];
    }
    float to = mx;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) to = fmaxf(to, m[j]);
    const float base = to == -__builtin_inff() ? 0.0f : to;
    const float f0 = __builtin_amdgcn_exp2f((mx - base) * a.c);
    mx = to;
    sum *= f0;
    o *= f0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j < n) {
        const float f = __builtin_amdgcn_exp2f((m[j] - base) * a.c);
        sum += l[j] * f;
        o += x[j] * f;
      }
  }
  if (!(finite(o[0]) && finite(o[1]) && finite(o[2]) && finite(o[3]))) {
    f32x4_t whole = {0, 0, 0, 0};  // as in join_row
#pragma unroll 1
    for (int i = 0; i < n; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float y = part[tile_of(i) * 4 * D][c];
        whole[c] += finite(y) ? 0.0f : y;
      }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (whole[c] != 0.0f) o[c] = whole[c];
  }
  const bool none = sum == 0.0f || quot(row, a.G) >= new_of(a, b);
  const u32x2 x = {none ? 0 : pack2(o[0] / sum, o[1] / sum),
                   none ? 0 : pack2(o[2] / sum, o[3] / sum)};
  *reinterpret_cast<u32x2*>(out_row(a, b, h, row) + 16 * group + 4 * g4) = x;
}

template <int D, int NT, typename DEAL>
int launch_join_many(const AttnArgs& a, hipStream_t st) {
  const int rows = a.S * a.G, block = 16 * NT * kWaves;
  const dim3 joins((unsigned)(a.B * a.Hk * a.rb), (unsigned)((std::min(rows, block) + 15) / 16),
                   (D / 16 + kWaves - 1) / kWaves);
  hipLaunchKernelGGL((join_many_kernel<D, NT, DEAL>), joins, dim3(kThreads), 0, st, a);
  return launch_status();
}

template <int D, typename DEAL>
int launch_join_few(const AttnArgs& a, hipStream_t st) {
  const dim3 joins((unsigned)(a.B * a.Hk), (unsigned)((a.S * a.G + kWaves - 1) / kWaves));
  hipLaunchKernelGGL((join_few_kernel<D, DEAL>), joins, dim3(kThreads), 0, st, a);
  return launch_status();
}

struct Shape {
  int nt;     // 0: attend_few_kernel; else row tiles of a wave of attend_many_kernel
  int block;  // rows of a workgroup
  int rb;     // row blocks
  int nwg;
};

// few: workgroups a CU holds of the kernel for up to 16 rows.
Shape shape_of(int64_t rows, int64_t D, int64_t cus, int few) {
  Shape s;
  s.nt = rows <= 16 ? 0 : rows <= 64 || D > 128 ? 1 : 2;
  s.block = s.nt ? 16 * s.nt * kWaves : 16;
  s.rb = (int)((rows + s.block - 1) / s.block);
  s.nwg = (int)(cus * (s.nt == 0 ? few : D <= 128 ? 2 : 1));
  return s;
}

int64_t workspace_of(const Shape& s, int64_t D) {
  return (int64_t)s.nwg * 2 * s.block * (D + 2) * 4;
}

bool head_dim_ok(int64_t D) { return D == 64 || D == 128 || D == 256; }

// Requests of up to `cap` keys that a call takes: the tiles of all are counted in 32 bits.
int64_t max_requests(int64_t S, int64_t Hq, int64_t Hk, int64_t D, int64_t cap) {
  if (S > (1 << 20) || Hq > (1 << 16) || S * Hq > 0x7fffffff || cap > ((int64_t)1 << 30)) return 0;
  const int64_t rb = shape_of(S * (Hq / Hk), D, 1, 1).rb;
  return std::min<int64_t>(0x7fffffff / (Hk * rb) / (cap / kStep + 8), 1 << 20);
}

// A call's arguments as the entry points get them; cache strides in elements.
struct AttnCall {
  const void *q, *k, *v;
  void* out;
  const int32_t *table, *kv_lens, *q_lens;
  int64_t B, S, Hq, Hk, D, q_sb, q_ss, q_sh, o_sb, o_ss, o_sh, c_sb, c_sh, c_ss;
  int64_t blocks, block_rows, table_ld, table_w, kv_len;
  int causal;
  float scale;
  int32_t* counters;
  void* workspace;
  int64_t workspace_bytes;
};

// The checks that entry points share, and the kernels' arguments.  1: nothing to do.
// chunk: elements of 16 bytes of the cache; few: as shape_of's.
int attn_args(const AttnCall& x, int chunk, int few, AttnArgs& a, Shape& s) {
  if (x.B < 0 || x.S < 0 || x.Hq < 0 || x.Hk < 0 || x.D <= 0 || x.blocks < 0 ||
      x.block_rows < 0 || x.workspace_bytes < 0)
    return UMIC_ERR_INVALID_ARG;
  if (x.B == 0 || x.S == 0 || x.Hq == 0) return 1;
  if (x.Hk == 0 || x.Hq % x.Hk || !(__builtin_fabsf(x.scale) <= 0x1p127f))
    return UMIC_ERR_INVALID_ARG;
  if (!x.q || !x.out || !x.workspace) return UMIC_ERR_INVALID_ARG;
  if (!head_dim_ok(x.D)) return UMIC_ERR_UNSUPPORTED;
  int64_t cap = x.block_rows;
  int shift = 30;
  if (x.table) {
    if (x.table_w < 0 || x.table_ld < x.table_w) return UMIC_ERR_INVALID_ARG;
    if (x.block_rows < 16 || (x.block_rows & (x.block_rows - 1))) return UMIC_ERR_UNSUPPORTED;
    if (x.table_w > ((int64_t)1 << 30) / x.block_rows) return UMIC_ERR_UNSUPPORTED;
    cap = x.blocks ? x.table_w * x.block_rows : 0;
    shift = __builtin_ctzll((unsigned long long)x.block_rows);
  } else if (x.blocks != x.B) {
    return UMIC_ERR_INVALID_ARG;
  }
  if (cap > 0 && (!x.k || !x.v)) return UMIC_ERR_INVALID_ARG;
  if (!x.kv_lens && (x.kv_len < 0 || x.kv_len > cap)) return UMIC_ERR_INVALID_ARG;
  if (((x.q_sb | x.q_ss | x.q_sh | x.o_sb | x.o_ss | x.o_sh) & 7) ||
      ((x.c_sb | x.c_sh | x.c_ss) & (chunk - 1)) || !aligned16(x.q) || !aligned16(x.k) ||
      !aligned16(x.v) || !aligned16(x.out) || !aligned16(x.workspace))
    return UMIC_ERR_UNSUPPORTED;
  const int64_t cus = device_cus();
  if (cus <= 0) return (int)hipErrorNoDevice;
  const int64_t G = x.Hq / x.Hk;
  if (x.B > max_requests(x.S, x.Hq, x.Hk, x.D, cap) || x.blocks > ((int64_t)1 << 30))
    return UMIC_ERR_UNSUPPORTED;
  s = shape_of(x.S * G, x.D, cus, few);
  if (x.workspace_bytes < workspace_of(s, x.D)) return UMIC_ERR_INVALID_ARG;
  if (x.c_ss < 0 || x.c_ss >= (1 << 24)) return UMIC_ERR_UNSUPPORTED;  // row offsets in a tile
  a.q = (const uint16_t*)x.q, a.k = (const uint16_t*)x.k, a.v = (const uint16_t*)x.v;
  a.out = (uint16_t*)x.out, a.table = x.table, a.kv_len = x.kv_lens, a.q_len = x.q_lens;
  a.counters = s.nwg > UMIC_ATTENTION_COUNTERS ? nullptr : x.counters;
  a.part = (float*)x.workspace;
  a.part_ml = a.part + (int64_t)s.nwg * 2 * s.block * x.D;
  a.q_sb = x.q_sb, a.q_ss = x.q_ss, a.q_sh = x.q_sh;
  a.o_sb = x.o_sb, a.o_ss = x.o_ss, a.o_sh = x.o_sh;
  a.c_sb = x.c_sb, a.c_sh = x.c_sh, a.c_ss = (int)x.c_ss, a.table_ld = x.table_ld;
  a.cap = (int)cap;
  a.B = (int)x.B, a.S = (int)x.S, a.Hk = (int)x.Hk, a.G = (int)G, a.rb = s.rb;
  a.len = x.kv_lens ? 0 : (int)x.kv_len, a.blocks = (int)x.blocks, a.shift = shift;
  a.nwg = s.nwg;
  // Many rows: two workgroups to a CU or one.  Between the two some CUs have twice the
  // others' work (128 tokens over 1024 keys: 288 workgroups 25 us, 256 of them 22).
  a.some = s.nt && a.nwg > cus ? (int)cus : a.nwg;
  a.causal = x.causal != 0;
  a.c = __builtin_fabsf(x.scale) * 1.4426950408889634f;
  if (a.c < 0x1p-126f) a.c = 0x1p-126f;  // masked scores are -inf: times 0 they would be NaN
  a.flip = x.scale < 0.0f ? 0x80008000u : 0u;
  return UMIC_OK;
}

// Bytes of workspace that a call takes; 0: of no such call.
int64_t workspace_bytes(int64_t S, int64_t Hq, int64_t Hk, int64_t D, int few) {
  if (S <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || !head_dim_ok(D) || S > (1 << 20) || Hq > (1 << 16))
    return 0;
  return workspace_of(shape_of(S * (Hq / Hk), D, device_cus(), few), D);
}

}  // namespace
}  // namespace umic
