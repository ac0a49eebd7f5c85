// Attention of a request's new tokens over its key / value cache, paged or
// contiguous:  o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max).
//
// The S new tokens' query heads that share a key head (G of them) are S G rows
// of one small product, packed in tiles of 16.  One pass over the keys: scores
// and output are v_mfma_f32_16x16x32_bf16 products with the keys as the left
// operand (S^T = K Q^T, O^T = V^T P^T), so that
//  * a lane's scores belong to one row (lane % 16), and so do its outputs: the
//    running maximum, the sum and the rescaling are lane-local, but for the
//    maximum over the four lanes of a row;
//  * the lane that computes keys 16 t + 4 g + i (t: key tile, g = lane / 16, i:
//    accumulator register) is the lane whose operand of the second product
//    holds them: p never leaves its registers;
//  * a key's row is read as the operand wants it, 16 bytes a lane; V is read
//    along its rows too, and turned in registers (v_perm of row pairs).
// p is split in two bf16 parts (p = hi + lo to 2^-17), each its own product: one
// rounding to bf16 would weigh as much as the output's own.
//
// Up to 16 rows (single tokens) the four waves of a workgroup take 32 keys each,
// and nothing goes through LDS until they are joined: HBM-bound.  More rows go
// 16 or 32 to a wave, and the waves share the keys through LDS.
//
// The key tiles of all requests, in one row, are dealt evenly over the launch's
// workgroups, so requests of all lengths fill the chip alike.  A workgroup that
// has a part of a request's tiles leaves (max, sum, output) in the workspace: at
// most two such parts each, of the first and the last of its segments.  They are
// joined in the order of the keys: by the workgroup that finishes last, for up
// to 16 rows and with counters to find that out, else by a second kernel.
//
// Measured, 32 query heads over 8 of 128: a token of two requests of 131001 keys each
// 173 us (6.2 TB/s), of 64 ragged requests up to 8192 keys 49 (5.1 TB/s), of one
// request of 3100 keys 9.9: 4 until its first keys are there, 1.7 for them, 3 to join
// 25 parts.  128 tokens over 65536 keys 233 us (590 TFLOP/s); four 128-token chunks
// 47, of which the second kernel takes 13 for 41 MB of parts.
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
template <int TILE, int LEAD, int LEAST>
struct Deal {
  unsigned each, more;
  int nwg;

  static __device__ __forceinline__ int tiles(int keys) { return (keys + TILE - 1) / TILE; }
  static __device__ __forceinline__ int units(int keys) {
    return keys > 0 ? tiles(keys) + LEAD : 0;
  }
  // most: that the chip holds; if that many have no work, no more than `some`
  __device__ __forceinline__ Deal(unsigned all, int most, int some) {
    const unsigned fit = (all + LEAST - 1) / LEAST;
    nwg = fit >= (unsigned)most ? most : min((int)fit, some);
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

  __device__ __forceinline__ void load_q(const AttnArgs& a, const Segment& s, int r0, int n16,
                                         int g4) {
    const int rows = a.S * a.G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = min(r0 + nt * 16 + n16, rows - 1);  // past them: computed, not written
      const int t = quot(r, a.G), g = r - t * a.G;
      lim[nt] = a.causal ? min(s.len, s.len - s.fresh + t + 1) : s.len;
      const uint16_t* qp =
          a.q + s.b * a.q_sb + (int64_t)(s.h * a.G + g) * a.q_sh + t * a.q_ss + g4 * 8;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        q[nt][kk] = *reinterpret_cast<const u32x4*>(qp + kk * 32) ^ a.flip;
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
  __device__ __forceinline__ void weights(const f32x4_t (&sc)[NT][2], float c, u32x4 (&ph)[NT],
                                          u32x4 (&pl)[NT]) {
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

// This workgroup's place in the deal: they go round the eight XCDs, and those of
// one XCD take neighbouring tiles.
__device__ __forceinline__ int dealt_wg(int nwg) {
  const int eighth = (nwg + 7) / 8;
  const int wg = (blockIdx.x & 7) * eighth + blockIdx.x / 8;
  return (int)(blockIdx.x / 8) < eighth && wg < nwg ? wg : -1;
}

// Up to 16 rows: a wave takes 32 of a tile's 128 keys.  The loads of a step are in
// flight while the one before is computed, and the next segment's first while the
// waves of this one are joined.
template <int D>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attend_few_kernel(AttnArgs a) {
  typedef Rows<D, 1, false> R;
  constexpr int KK = R::KK, DV = R::DV, VW = R::VW;
  constexpr int LDR = D + 4;  // row of the join's LDS, in floats
  constexpr int kTile = kStep * kWaves;
  __shared__ int sums[kWaves];
  __shared__ int found[2];
  __shared__ int arrived[2];
  __shared__ Segment kept[2];  // those that other workgroups have a part of: the first, the last
  __shared__ float ml[kWaves][16][2];
  __shared__ float acc_lds[kWaves][16][LDR];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;

  Scan scan = {};
  const int even = a.kv_len ? 0 : FewDeal::units(a.len);  // units of each, if all have as many
  if (a.kv_len)
    scan = scan_units<FewDeal>(a, sums);
  else
    scan.all = even * a.B;
  const FewDeal deal((unsigned)(scan.all * a.Hk), a.nwg, a.some);
  const int wg = dealt_wg(deal.nwg);
  const int rows = a.S * a.G;
  if (wg >= 0) {
    Walk<FewDeal, false> walk;
    walk.start(a, deal, scan, even, wg, found);
    R r;
    Segment seg, nxt;
    int split = 0;  // bits: which of `kept` there are
    Place here;
    u32x4 kf[2][KK];
    uint32_t vr[R::VR];
    // rows that are not there are read again from one that is
    auto load_k = [&](const AttnArgs& a, const Place& p) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t* kp = a.k + p.at[i];
        const unsigned off = __umul24(min(n16, max(p.n[i] - 1, 0)), a.c_ss) + g4 * 8;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kf[i][kk] = ld_stream(reinterpret_cast<const u32x4*>(kp + off + kk * 32));
      }
    };
    auto load_v = [&](const AttnArgs& a, const Place& p) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2;
        const unsigned off =
            __umul24(min(4 * g4 + (j & 3), max(p.n[i] - 1, 0)), a.c_ss) + n16 * DV;
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(a.v + p.at[i] + off);
#pragma unroll
        for (int w = 0; w < VW; ++w) vr[j * VW + w] = vp[w];
      }
    };
    auto first_of = [&](const AttnArgs& a, const Segment& s) {
      const Keys keys = keys_of(a, s);
      const int k0 = s.t0 * kTile + wave * kStep;
      return place_of(a, keys, k0, blocks_of(a, keys, k0));
    };
    walk.next(a, seg);  // a dealt workgroup has one
    here = first_of(a, seg);
    load_k(a, here);
    load_v(a, here);
    r.load_q(a, seg, 0, n16, g4);
    for (bool go = true; go;) {
      go = walk.next(args_again(), nxt);
      const Place turn = go ? first_of(args_again(), nxt) : here;
      bool turned = false;  // the next segment's keys are on their way
      const Keys keys = keys_of(args_again(), seg);
      r.clear();
      for (int t = seg.t0; t < seg.t1; ++t) {
        const int k0 = t * kTile + wave * kStep, k1 = k0 + kTile;
        if (k0 >= r.hi) break;
        const bool more = t + 1 < seg.t1 && k1 < r.hi;
        Place next = turn;
        if (more) next = place_of(a, keys, k1, blocks_of(a, keys, k1));
        turned = !more;
        f32x4_t sc[1][2];
        r.scores(kf, sc);
        if (more || go) load_k(a, next);  // under the softmax and the second product
        const bool edge = k0 + kStep > r.lo || here.n[0] < 16 || here.n[1] < 16;
        if (edge) r.mask(sc, vr, here.n, k0, g4);
        u32x4 ph[1], pl[1];
        r.weights(sc, a.c, ph, pl);
        if (edge && r.lo < seg.len) r.hide(vr, a, here, k0, g4);
        r.product(vr, ph, pl);
        if (more || go) load_v(a, next);
        here = next;
      }
      if (go) {
        if (!turned) {
          load_k(a, turn);
          load_v(a, turn);
        }
        here = turn;
        r.load_q(args_again(), nxt, 0, n16, g4);
      }

      // join the waves
      const AttnArgs args = args_again();
      const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
      const int slot = wg * 2 + (seg.t0 == 0 ? 1 : 0);
      r.l[0] += __shfl_xor(r.l[0], 16, kWave);
      r.l[0] += __shfl_xor(r.l[0], 32, kWave);
      if (g4 == 0) {
        ml[wave][n16][0] = r.max_of(0);
        ml[wave][n16][1] = r.l[0];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DV; ++e) acc_lds[wave][n16][(4 * g4 + i) * DV + e] = r.acc[0][e][i];
      __syncthreads();
      // thread: row tid / 16, columns DV (tid % 16) ..
      const int rr = threadIdx.x >> 4, col = (threadIdx.x & 15) * DV;
      if (rr < rows) {
        float mx = ml[0][rr][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, ml[w][rr][0]);
        const float base = mx == -__builtin_inff() ? 0.0f : mx;
        f32x4_t o[DV / 4] = {};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f((ml[w][rr][0] - base) * args.c);
          sum += ml[w][rr][1] * f;
#pragma unroll
          for (int e = 0; e < DV; ++e) o[e / 4][e % 4] += acc_lds[w][rr][col + e] * f;
        }
        const int token = quot(rr, args.G);
        const int lim = args.causal ? seg.len - seg.fresh + token + 1 : seg.len;
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
        if (threadIdx.x == 0) kept[seg.t0 == 0 ? 1 : 0] = seg;
      }
      __syncthreads();  // LDS is used again
      seg = nxt;
    }
    const AttnArgs args = args_again();
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
        deal.holders(uniform(kept[i].at), uniform(kept[i].tiles), w0[i], w1[i]);
        if (threadIdx.x == 0)
          arrived[i] = __hip_atomic_fetch_add(args.counters + w0[i], 1, __ATOMIC_RELAXED,
                                              __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int v0 = i ? w0[1] : w0[0], v1 = i ? w1[1] : w1[0];
        // others' parts are missing
        if (!(split >> i & 1) || uniform(arrived[i]) != v1 - v0) continue;
        if (threadIdx.x == 0) args.counters[v0] = 0;  // for the next call
        const int b = uniform(kept[i].b), h = uniform(kept[i].h), fresh = uniform(kept[i].fresh);
        for (int row = wave; row < rows; row += kWaves)
          join_row<D, true>(args, v0, v1, row, quot(row, args.G) >= fresh,
                            out_row(args, b, h, row));
      }
    }
  }
  const AttnArgs z = args_again();
  if (z.counters) zero_rows<D>(z);
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

// 16 bytes of each lane, from base + off (bytes), to 1 KB of LDS at `to`.  Written
// out: before any LDS read the compiler waits for all loads into LDS that it knows
// of, those of the steps to come included.  Its own counts of loads in flight stay
// safe, as more are in flight than it counts; nothing is written to a register.
// The wait states: of m0 (1), and of scalars that a vector instruction wrote (5),
// which the compiler does not see to inside the block.  (With the builtin every step
// waited for the loads of the steps to come: four 128-token chunks took 1.7 times as
// long.)
__device__ __forceinline__ void load_to_lds(const void* base, unsigned off, unsigned to) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(to), "v"(off), "s"(base)
               : "memory");
}

// More rows: each wave has 16 NT of the workgroup's 64 NT, and the keys go through
// a ring in LDS, kRing - 1 steps of 32 on their way: the loads take a few
// thousand cycles (with one step ahead, through registers, four 128-token chunks
// took 12% longer).  A row's 16-byte chunks are permuted so that neither the reads
// of a chunk down the rows (K: ^ row) nor those of two chunks of eight rows (V: ^ 2
// row) meet in a bank.
// What bounds it: of a step's 3900 cycles for two waves of a SIMD the matrix
// instructions take 1540 (48 a wave, the second product twice) and the vector ones
// 1800 (177 a wave, 16 of them exponentials), which run beside the former for a
// quarter of their time.  Matrix and vector instructions in turn, priorities, the
// next K read early, a barrier for two steps, eight waves that halve the parts: none
// was faster (128 tokens over 65536 keys stayed within 2%, the last cost the chunks
// 7 us).
template <int D, int NT>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attend_many_kernel(AttnArgs a) {
  typedef Rows<D, NT, true> R;
  constexpr int KK = R::KK, DV = R::DV;
  constexpr int CH = D / 8;                   // chunks of a row
  constexpr int PER = kStep * CH / kThreads;  // chunks of K (and V) a thread moves a step
  constexpr int kBlock = 16 * NT * kWaves;    // rows of a workgroup
  constexpr int kRing = 4;
  constexpr int LOADS = 2 * PER;  // of a wave, a step
  __shared__ int sums[kWaves];
  __shared__ int found[2];
  __shared__ u32x4 kv[kRing][2][kStep * CH];  // [slot][K, V]
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;
  auto k_swizzle = [](int row) { return CH >= 16 ? row & 15 : (row >> 1) & 7; };
  auto v_swizzle = [](int row) { return CH >= 16 ? (row & 7) * 2 : ((row >> 1) & 3) * 2; };

  Scan scan = {};
  const int even = a.kv_len ? 0 : ManyDeal::units(a.len);
  if (a.kv_len)
    scan = scan_units<ManyDeal>(a, sums);
  else
    scan.all = even * a.B;
  const ManyDeal deal((unsigned)(scan.all * a.Hk * a.rb), a.nwg, a.some);
  const int wg = dealt_wg(deal.nwg);
  const int rows = a.S * a.G;
  if (wg < 0) return;
  Walk<ManyDeal, true> walk;
  walk.start(a, deal, scan, even, wg, found);
  R r;
  Segment seg;
  // A load instruction fills 64 neighbouring cells of LDS: which chunk a lane
  // fetches follows from its cell.  Rows that are not there are another's again.
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_void*)kv) +
                       wave * kWave * 16;
  auto fetch = [&](const AttnArgs& a, int slot, const Place& p) {
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      const int c = x * kThreads + (int)threadIdx.x, row = c / CH;
      const int i = (CH >= 16 ? x * (kThreads / CH) : wave * (kWave / CH)) >> 4;  // its tile
      const int n = i ? p.n[1] : p.n[0];
      const int64_t at = i ? p.at[1] : p.at[0];
      const unsigned off = __umul24(min(row & 15, max(n - 1, 0)), a.c_ss) * 2;
      const unsigned to = lds + (slot * 2 * kStep * CH + x * kThreads) * 16;
      load_to_lds(a.k + at, off + ((c % CH) ^ k_swizzle(row)) * 16, to);
      load_to_lds(a.v + at, off + ((c % CH) ^ v_swizzle(row)) * 16, to + kStep * CH * 16);
    }
  };
  while (walk.next(args_again(), seg)) {
    const AttnArgs a = args_again();
    const int r0 = seg.rb * kBlock + wave * 16 * NT;
    // the block's last key that any row sees
    int end = seg.len;
    if (a.causal)
      end = min(end, seg.len - seg.fresh + quot(min((seg.rb + 1) * kBlock, rows) - 1, a.G) + 1);
    const int t1 = min(seg.t1, (max(end, 0) + kStep - 1) / kStep);
    const Keys keys = keys_of(a, seg);
    auto blocks = [&](int t) { return blocks_of(a, keys, t * kStep); };
    Blocks ahead[kRing];
    unsigned full = 0;  // bit t % 32: step t's pages are all there
    auto send = [&](int t, const Blocks& x) {
      const Place p = place_of(a, keys, t * kStep, x);
      fetch(a, t % kRing, p);
      const unsigned bit = 1u << (t & 31);
      full = p.n[0] == 16 && p.n[1] == 16 ? full | bit : full & ~bit;
    };
    landed_barrier<63>();  // the last segment's reads are done
#pragma unroll
    for (int i = 0; i < kRing; ++i) ahead[i] = blocks(seg.t0 + i);
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i)
      if (seg.t0 + i < t1) send(seg.t0 + i, ahead[i]);
    Blocks later = ahead[kRing - 1];
    r.load_q(args_again(), seg, r0, n16, g4);
    r.clear();
    for (int t = seg.t0; t < t1; ++t) {
      const int k0 = t * kStep;
      // this step's keys are there, those of the step before have been read
      if (t + kRing - 2 < t1)
        landed_barrier<(kRing - 2) * LOADS>();
      else if (t + 1 < t1 && kRing == 4)
        landed_barrier<LOADS>();
      else
        landed_barrier<0>();
      const bool idle = k0 >= r.hi || r0 >= rows;
      const u32x4* const ks = kv[t % kRing][0];
      const u32x4* const vs = kv[t % kRing][1];
      u32x4 kf[2][KK];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kf[i][kk] = ks[(16 * i + n16) * CH + ((kk * 4 + g4) ^ k_swizzle(n16))];
      if (t + kRing - 1 < t1) {
        send(t + kRing - 1, later);
        later = blocks(t + kRing);
      }
      if (idle) continue;
      f32x4_t sc[NT][2];
      r.scores(kf, sc);
      // a read that turns 4 keys by 16 columns over 16 lanes: lane n16 gives the
      // address of 4 columns of a key and gets one column of the 4 keys
      uint32_t vr[R::VR];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 16 * i + 4 * g4 + (n16 >> 2);
#pragma unroll
        for (int e = 0; e < DV; ++e) {
          const u32x4* const c = vs + row * CH + ((2 * e + ((n16 >> 1) & 1)) ^ v_swizzle(row));
          const uint64_t x = __builtin_bit_cast(
              uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s16x4*)(reinterpret_cast<const uint64_t*>(c) + (n16 & 1))));
          vr[4 * e + 2 * i] = (uint32_t)x;
          vr[4 * e + 2 * i + 1] = (uint32_t)(x >> 32);
        }
      }
      const bool edge = k0 + kStep > r.lo || !(full >> (t & 31) & 1);
      Place here = {};
      if (edge) {
        here = place_of(a, keys, k0, blocks(t));
        r.mask(sc, vr, here.n, k0, g4);
      }
      u32x4 ph[NT], pl[NT];
      r.weights(sc, a.c, ph, pl);
      if (edge && r.lo < seg.len) r.hide(vr, a, here, k0, g4);
      r.product(vr, ph, pl);
    }
    const AttnArgs args = args_again();
    const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
    const int slot = wg * 2 + (seg.t0 == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum = r.l[nt];
      sum += __shfl_xor(sum, 16, kWave);
      sum += __shfl_xor(sum, 32, kWave);
      const int row = r0 + nt * 16 + n16;
      const bool padded = quot(row, args.G) >= seg.fresh;
      restore<DV, 16>(r.acc[nt], !padded && sum == sum, args, keys_of(args, seg), seg.t0 * kStep,
                      t1 * kStep, r.lim[nt], 4 * g4);
      if (row >= rows) continue;
      // a lane's columns: 16 e + 4 g4 .. + 4
      if (whole) {
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
        const int64_t tile = (int64_t)slot * (kBlock / 16) + wave * NT + nt;
        f32x4_t* p = reinterpret_cast<f32x4_t*>(args.part) + tile * 4 * D + lane;
#pragma unroll
        for (int e = 0; e < DV; ++e) p[e * kWave] = r.acc[nt][e];
        if (g4 == 0) {
          args.part_ml[(tile * 16 + n16) * 2] = r.max_of(nt);
          args.part_ml[(tile * 16 + n16) * 2 + 1] = sum;
        }
      }
    }
  }
}

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
template <int D>
__global__ __launch_bounds__(kThreads) void join_few_kernel(AttnArgs a) {
  __shared__ int sums[kWaves];
  __shared__ int found;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int b = blockIdx.x / a.Hk, h = blockIdx.x - b * a.Hk;
  int w0, w1;
  const bool any = find_parts<FewDeal>(a, b, h, sums, &found, w0, w1);
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
template <int D, int NT>
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
  const bool any = find_parts<ManyDeal>(a, b, pair, sums, &found, w0, w1);
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

struct Shape {
  int nt;     // 0: attend_few_kernel; else row tiles of a wave of attend_many_kernel
  int block;  // rows of a workgroup
  int rb;     // row blocks
  int nwg;
};

Shape shape_of(int64_t rows, int64_t D, int64_t cus) {
  Shape s;
  s.nt = rows <= 16 ? 0 : rows <= 64 || D > 128 ? 1 : 2;
  s.block = s.nt ? 16 * s.nt * kWaves : 16;
  s.rb = (int)((rows + s.block - 1) / s.block);
  s.nwg = (int)(cus * (D <= 128 ? 2 : 1));
  return s;
}

int64_t workspace_of(const Shape& s, int64_t D) {
  return (int64_t)s.nwg * 2 * s.block * (D + 2) * 4;
}

template <int D, int NT>
int launch_many(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.nwg + 7) / 8 * 8)), threads(kThreads);
  hipLaunchKernelGGL((attend_many_kernel<D, NT>), grid, threads, 0, st, a);
  if (const int e = launch_status()) return e;
  const int rows = a.S * a.G, block = 16 * NT * kWaves;
  const dim3 joins((unsigned)(a.B * a.Hk * a.rb), (unsigned)((std::min(rows, block) + 15) / 16),
                   (D / 16 + kWaves - 1) / kWaves);
  hipLaunchKernelGGL((join_many_kernel<D, NT>), joins, threads, 0, st, a);
  return launch_status();
}

template <int D>
int launch(const Shape& s, const AttnArgs& a, hipStream_t st) {
  if constexpr (D <= 128)
    if (s.nt == 2) return launch_many<D, 2>(a, st);
  if (s.nt) return launch_many<D, 1>(a, st);
  const dim3 grid((unsigned)((a.nwg + 7) / 8 * 8)), threads(kThreads);
  hipLaunchKernelGGL((attend_few_kernel<D>), grid, threads, 0, st, a);
  const int e = launch_status();
  if (e || a.counters) return e;
  const dim3 joins((unsigned)(a.B * a.Hk), (unsigned)((a.S * a.G + kWaves - 1) / kWaves));
  hipLaunchKernelGGL((join_few_kernel<D>), joins, threads, 0, st, a);
  return launch_status();
}

bool head_dim_ok(int64_t D) { return D == 64 || D == 128 || D == 256; }

// Requests of up to `cap` keys that a call takes: the tiles of all are counted in 32 bits.
int64_t max_requests(int64_t S, int64_t Hq, int64_t Hk, int64_t D, int64_t cap) {
  if (S > (1 << 20) || Hq > (1 << 16) || S * Hq > 0x7fffffff || cap > ((int64_t)1 << 30)) return 0;
  const int64_t rb = shape_of(S * (Hq / Hk), D, 1).rb;
  return std::min<int64_t>(0x7fffffff / (Hk * rb) / (cap / kStep + 8), 1 << 20);
}

}  // namespace
}  // namespace umic

extern "C" int64_t umic_cache_attention_workspace_bytes(int64_t S, int64_t Hq, int64_t Hk,
                                                        int64_t D) {
  using namespace umic;
  if (S <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || !head_dim_ok(D) || S > (1 << 20) || Hq > (1 << 16))
    return 0;
  return workspace_of(shape_of(S * (Hq / Hk), D, device_cus()), D);
}

extern "C" int64_t umic_cache_attention_max_requests(int64_t S, int64_t Hq, int64_t Hk, int64_t D,
                                                     int64_t cap) {
  using namespace umic;
  if (S <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || !head_dim_ok(D) || cap < 0) return 0;
  return max_requests(S, Hq, Hk, D, cap);
}

extern "C" int umic_cache_attention_bf16(
    const void* q, const void* k, const void* v, void* out, const int32_t* table,
    const int32_t* kv_lens, const int32_t* q_lens, int64_t B, int64_t S, int64_t Hq, int64_t Hk,
    int64_t D, int64_t q_sb, int64_t q_ss, int64_t q_sh, int64_t o_sb, int64_t o_ss, int64_t o_sh,
    int64_t c_sb, int64_t c_sh, int64_t c_ss, int64_t blocks, int64_t block_rows, int64_t table_ld,
    int64_t table_w, int64_t kv_len, int causal, float scale, int32_t* counters,
    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace umic;
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || blocks < 0 || block_rows < 0 ||
      workspace_bytes < 0)
    return UMIC_ERR_INVALID_ARG;
  if (B == 0 || S == 0 || Hq == 0) return UMIC_OK;
  if (Hk == 0 || Hq % Hk || !(__builtin_fabsf(scale) <= 0x1p127f))
    return UMIC_ERR_INVALID_ARG;
  if (!q || !out || !workspace) return UMIC_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return UMIC_ERR_UNSUPPORTED;
  int64_t cap = block_rows;
  int shift = 30;
  if (table) {
    if (table_w < 0 || table_ld < table_w) return UMIC_ERR_INVALID_ARG;
    if (block_rows < 16 || (block_rows & (block_rows - 1))) return UMIC_ERR_UNSUPPORTED;
    if (table_w > ((int64_t)1 << 30) / block_rows) return UMIC_ERR_UNSUPPORTED;
    cap = blocks ? table_w * block_rows : 0;
    shift = __builtin_ctzll((unsigned long long)block_rows);
  } else if (blocks != B) {
    return UMIC_ERR_INVALID_ARG;
  }
  if (cap > 0 && (!k || !v)) return UMIC_ERR_INVALID_ARG;
  if (!kv_lens && (kv_len < 0 || kv_len > cap)) return UMIC_ERR_INVALID_ARG;
  if (((q_sb | q_ss | q_sh | o_sb | o_ss | o_sh | c_sb | c_sh | c_ss) & 7) || !aligned16(q) ||
      !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace))
    return UMIC_ERR_UNSUPPORTED;
  const int64_t cus = device_cus();
  if (cus <= 0) return (int)hipErrorNoDevice;
  const int64_t G = Hq / Hk;
  if (B > max_requests(S, Hq, Hk, D, cap) || blocks > ((int64_t)1 << 30))
    return UMIC_ERR_UNSUPPORTED;
  const Shape s = shape_of(S * G, D, cus);
  if (workspace_bytes < workspace_of(s, D)) return UMIC_ERR_INVALID_ARG;
  if (s.nwg > UMIC_ATTENTION_COUNTERS) counters = nullptr;
  if (c_ss < 0 || c_ss >= (1 << 24)) return UMIC_ERR_UNSUPPORTED;  // row offsets in a tile
  AttnArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.out = (uint16_t*)out, a.table = table, a.kv_len = kv_lens, a.q_len = q_lens;
  a.counters = counters;
  a.part = (float*)workspace;
  a.part_ml = a.part + (int64_t)s.nwg * 2 * s.block * D;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.o_sb = o_sb, a.o_ss = o_ss, a.o_sh = o_sh;
  a.c_sb = c_sb, a.c_sh = c_sh, a.c_ss = (int)c_ss, a.table_ld = table_ld, a.cap = (int)cap;
  a.B = (int)B, a.S = (int)S, a.Hk = (int)Hk, a.G = (int)G, a.rb = s.rb;
  a.len = kv_lens ? 0 : (int)kv_len, a.blocks = (int)blocks, a.shift = shift;
  // Single tokens of a few segments, up to a quarter of the CUs': a workgroup to a
  // CU.  The second hides the starts and ends of segments; with few it only doubles
  // their parts (8 segments of 12288 keys 18 us for 25, 64 of 1024 14.5 for 15.4; 128
  // of 300 15.2 for 13.6, 64 ragged requests 74 for 60).
  a.nwg = s.nt == 0 && B * Hk * 4 <= cus ? (int)cus : s.nwg;
  // Many rows: two workgroups to a CU or one.  Between the two some CUs have twice the
  // others' work (128 tokens over 1024 keys: 288 workgroups 25 us, 256 of them 22).
  a.some = s.nt && a.nwg > cus ? (int)cus : a.nwg;
  a.causal = causal != 0;
  a.c = __builtin_fabsf(scale) * 1.4426950408889634f;
  if (a.c < 0x1p-126f) a.c = 0x1p-126f;  // masked scores are -inf: times 0 they would be NaN
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  hipStream_t st = as_stream(stream);
  if (D == 64) return launch<64>(s, a, st);
  if (D == 128) return launch<128>(s, a, st);
  return launch<256>(s, a, st);
}
