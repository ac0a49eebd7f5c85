// Rotary rows as the kernels that write them share it: from positions of several axes,
// in bf16 (axial.hip), and beside codes of 8 bits (cache8.hip).
#pragma once

#include "common.hpp"
#include "gemm_ks.hpp"  // device_cus

namespace umic {
namespace {

constexpr int kThreads = 256;
// Pairs of chunks a thread has in flight: 2, and 3 where the norm's sums make a
// round longer (16381 tokens without: 68.5 us, 71 with 3; 3100 with it: 17.9, 19.6
// with 2).
template <bool NORM>
constexpr int kItemsOf = NORM ? 3 : 2;
constexpr int kMaxTokens = 16;   // of a workgroup
constexpr int kMaxHalf = 256;    // D/2 of the largest head

struct AxialArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* qo;
  uint16_t* ko;  // rows, or pages (slots)
  uint16_t* vo;
  const int64_t* positions;
  const uint64_t* turn;
  const int32_t* axis;
  const int64_t* slots;
  const uint16_t* qw;
  const uint16_t* kw;
  int64_t T, Hq, Hk, D, A;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh;
  int64_t ko_sb, ko_sh, ko_st;  // block, head, row (no slots: token ko_st)
  int64_t p_sa, p_st, slots_n;
  int shift;
  float eps, scale;
  int tokens;       // of a workgroup
  SmallDiv group;   // lanes of a head row
  SmallDiv rows;    // head rows of a token
  SmallDiv half;    // D / 2
};

// Sine and cosine of a position's angle, turn being 64-bit fractions of a turn.  FINE: of
// its distance from the nearest quarter turn, whose rounding to fp32 is 2^-25 of at most
// pi / 4 and not of pi.
template <bool FINE>
__device__ __forceinline__ void turn_of(int64_t pos, uint64_t turn, float& s, float& c) {
  const int32_t frac = (int32_t)(((uint64_t)pos * turn) >> 32);
  if constexpr (FINE) {
    const int32_t quarter = (int32_t)(((uint32_t)frac + 0x20000000u) >> 30);
    const int32_t rest = (int32_t)((uint32_t)frac - ((uint32_t)quarter << 30));
    float x, y;
    sincospif((float)rest * 0x1p-31f, &x, &y);
    const float p = quarter & 1 ? y : x, q = quarter & 1 ? x : y;
    s = quarter & 2 ? -p : p;
    c = (quarter + 1) & 2 ? -q : q;
  } else {
    sincospif((float)frac * 0x1p-31f, &s, &c);
  }
}

// VEC elements as they lie in memory
template <int VEC>
struct Raw;
template <>
struct Raw<8> {
  u32x4 v;
  __device__ __forceinline__ void load(const uint16_t* p) {
    v = ld_stream(reinterpret_cast<const u32x4*>(p));
  }
  template <bool NT>
  __device__ __forceinline__ void store(uint16_t* p) const {
    if constexpr (NT)
      st_stream(reinterpret_cast<u32x4*>(p), v);
    else
      *reinterpret_cast<u32x4*>(p) = v;
  }
  __device__ __forceinline__ void unpack(float* f) const { unpack8(v, f); }
  __device__ __forceinline__ void pack(const float* f) { v = pack8(f); }
};
template <>
struct Raw<4> {
  u32x2 v;
  __device__ __forceinline__ void load(const uint16_t* p) {
    v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
  }
  template <bool NT>
  __device__ __forceinline__ void store(uint16_t* p) const {
    *reinterpret_cast<u32x2*>(p) = v;
  }
  __device__ __forceinline__ void unpack(float* f) const { unpack4(v, f); }
  __device__ __forceinline__ void pack(const float* f) { v = pack4(f); }
};

// Where the (cos, sin) of a token's pair lies among its D floats, if lanes of 8 pairs each
// are to read theirs 16 bytes at a time side by side: [two pairs of a lane][lane].  (Pair by
// pair, 64 bytes a lane, the reads met in their banks: 16381 tokens of 32 + 8 heads with
// 8-bit rows 70 us for 63.)
__device__ __forceinline__ int turn_at(int pair, int lanes) {
  return ((pair >> 1 & 3) * lanes + (pair >> 3)) * 4 + (pair & 1) * 2;
}

// A lane holds VEC elements of each half of a head row; `group` lanes (a power
// of two with the norm, whose sum runs over them; lanes past the row idle) hold
// a row.  NT: stores past the caches, where the halves of a row are whole lines
// (16381 tokens of 32 + 8 heads of 128: 72 us for 80; rows of 80, which are not,
// 46 for 40).
// block: of a.tokens tokens; cs: [token][pair] (cos, sin) in LDS.  FINE: turn_of's, and
// turn_at's order (VEC 8).
template <int VEC, bool NORM, bool NT, bool FINE = false>
__device__ __forceinline__ void axial_rows(const AxialArgs& a, unsigned block, float* cs) {
  constexpr int kItems = kItemsOf<NORM>;
  const int half = a.half.d;
  const int64_t t0 = (int64_t)block * a.tokens;
  const int here = (int)(a.T - t0 < a.tokens ? a.T - t0 : a.tokens);
  const int items = here * a.rows.d * a.group.d;
  Raw<VEC> lo[kItems], hi[kItems];
  uint16_t* dst[kItems];  // NULL: not written
  int at[kItems];         // token and pair
  int kind[kItems];       // 0 q, 1 k, 2 v
  auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int i = base + u * kThreads + (int)threadIdx.x;
      int c, h;
      const int row = div_small(a.group, i < items ? i : 0, c);
      const int t = div_small(a.rows, row, h);
      const bool active = i < items && c * VEC < half;
      const int64_t tok = t0 + t;
      kind[u] = h < a.Hq ? 0 : h < a.Hq + a.Hk ? 1 : 2;
      const uint16_t* src;
      dst[u] = nullptr;
      const int d = active ? c * VEC : 0;
      if (kind[u] == 0) {
        src = a.q + tok * a.q_st + h * a.q_sh;
        if (active) dst[u] = a.qo + tok * a.qo_st + h * a.qo_sh + d;
      } else {
        const int hk = h - (int)a.Hq - (kind[u] == 2 ? (int)a.Hk : 0);
        src = kind[u] == 1 ? a.k + tok * a.k_st + hk * a.k_sh : a.v + tok * a.v_st + hk * a.v_sh;
        uint16_t* out = kind[u] == 1 ? a.ko : a.vo;
        if (!a.slots) {
          if (active) dst[u] = out + tok * a.ko_st + hk * a.ko_sh + d;
        } else {  // a slot outside the pool is not written
          const int64_t slot = a.slots[tok];
          const int64_t page = slot >> a.shift, r = slot & (((int64_t)1 << a.shift) - 1);
          if (active && slot >= 0 && slot < a.slots_n)
            dst[u] = out + page * a.ko_sb + hk * a.ko_sh + r * a.ko_st + d;
        }
      }
      at[u] = FINE ? t * 2 * half + (d >> 1) : t * half + d;
      lo[u].load(src + d);
      hi[u].load(src + half + d);
    }
  };
  // with the norm `group` divides the workgroup: a thread's chunk is always the same
  const int c0 = NORM ? (int)threadIdx.x & (a.group.d - 1) : 0;
  load(0);
  for (int i = threadIdx.x; i < here * half; i += kThreads) {
    int f;
    const int t = div_small(a.half, i, f);
    const int ax = a.axis[f];
    float s = 0.0f, c = 1.0f;
    if (ax >= 0 && ax < a.A) {  // an axis that is not there does not turn
      const int64_t pos = a.positions[ax * a.p_sa + (t0 + t) * a.p_st];
      turn_of<FINE>(pos, a.turn[f], s, c);
    }
    const int to = FINE ? t * 2 * half + turn_at(f, half >> 3) : 2 * i;
    cs[to] = c * a.scale;
    cs[to + 1] = s * a.scale;
  }
  __syncthreads();
  for (int base = 0; base < items; base += kItems * kThreads) {
    if (base) load(base);
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (base + u * kThreads >= items) break;  // whole waves: the norm's sums need theirs
      if (kind[u] == 2) {
        if (dst[u]) {
          lo[u].template store<NT>(dst[u]);
          hi[u].template store<NT>(dst[u] + half);
        }
        continue;
      }
      float x[VEC], y[VEC], ox[VEC], oy[VEC];
      lo[u].unpack(x);
      hi[u].unpack(y);
      const int t = at[u];
      if constexpr (NORM) {
        float ss = 0.0f;
        if (c0 * VEC < half)
#pragma unroll
          for (int j = 0; j < VEC; ++j) ss += x[j] * x[j] + y[j] * y[j];
        for (int m = 1; m < a.group.d; m <<= 1) ss += __shfl_xor(ss, m, kWave);
        const float r = rsqrt_cr(ss / (float)a.D + a.eps);
        // read here, from the cache: held from the start they cost a wave of occupancy
        // (3100 tokens 19.9 us for 18.2)
        const uint16_t* w = (kind[u] == 0 ? a.qw : a.kw) + (c0 * VEC < half ? c0 * VEC : 0);
        typedef decltype(lo[u].v) vec_t;
        Raw<VEC> w0, w1;
        w0.v = *reinterpret_cast<const vec_t*>(w);
        w1.v = *reinterpret_cast<const vec_t*>(w + half);
        float wx[VEC], wy[VEC];
        w0.unpack(wx);
        w1.unpack(wy);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[j] = x[j] * r * wx[j];
          y[j] = y[j] * r * wy[j];
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int from = FINE ? t + (j >> 1) * (half >> 1) + (j & 1) * 2 : 2 * (t + j);
        const float co = cs[from], si = cs[from + 1];
        ox[j] = x[j] * co - y[j] * si;
        oy[j] = y[j] * co + x[j] * si;
      }
      if (dst[u]) {
        Raw<VEC> o;
        o.pack(ox);
        o.template store<NT>(dst[u]);
        o.pack(oy);
        o.template store<NT>(dst[u] + half);
      }
    }
  }
}

// How a launch is shaped: elements of a lane's load, workgroups, stores past the caches.
struct AxialShape {
  int vec;
  unsigned blocks;
  size_t lds;
  bool lines;
};

// Fills what the kernel divides by.
int axial_shape(AxialArgs& a, AxialShape& s) {
  const bool norm = a.qw != nullptr;
  int64_t low = a.q_st | a.q_sh | a.k_st | a.k_sh | a.qo_st | a.qo_sh | a.ko_st | a.ko_sh;
  uintptr_t ptr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.qo | (uintptr_t)a.ko |
                  (uintptr_t)a.qw | (uintptr_t)a.kw;
  if (a.slots) {
    low |= a.v_st | a.v_sh | a.ko_sb;
    ptr |= (uintptr_t)a.v | (uintptr_t)a.vo;
  }
  const int64_t half = a.D / 2;
  int vec;
  if (half % 8 == 0 && !(low & 7) && !(ptr & 15))
    vec = 8;
  else if (half % 4 == 0 && !(low & 3) && !(ptr & 7))
    vec = 4;
  else
    return UMIC_ERR_UNSUPPORTED;
  int64_t group = half / vec;
  if (norm)
    while (group & (group - 1)) ++group;
  const int64_t rows = a.Hq + a.Hk * (a.slots ? 2 : 1), per = rows * group;
  if (group > kWave || per * kMaxTokens >= (1 << 22)) return UMIC_ERR_UNSUPPORTED;
  a.group = small_div((int)group);
  a.rows = small_div((int)rows);
  a.half = small_div((int)half);
  // as many tokens as one round of loads covers, fewer where the chip is not full
  const int64_t cus = device_cus();
  int64_t tokens = (norm ? kItemsOf<true> : kItemsOf<false>) * kThreads / per;
  if (cus > 0 && tokens > (a.T + 2 * cus - 1) / (2 * cus)) tokens = (a.T + 2 * cus - 1) / (2 * cus);
  a.tokens = (int)(tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens);
  const int64_t blocks = (a.T + a.tokens - 1) / a.tokens;
  if (blocks > 0x7fffffff) return UMIC_ERR_UNSUPPORTED;
  s = AxialShape{vec, (unsigned)blocks, (size_t)a.tokens * half * 2 * sizeof(float),
                 half % 64 == 0};
  return UMIC_OK;
}

// The checks both entry points share; 1: nothing to do.
int check_axial(const AxialArgs& a) {
  if (a.T < 0 || a.Hq < 0 || a.Hk < 0 || a.D <= 0 || a.A <= 0) return UMIC_ERR_INVALID_ARG;
  if (a.T == 0 || a.Hq + a.Hk == 0) return 1;
  if ((a.Hq && (!a.q || !a.qo)) || (a.Hk && (!a.k || !a.ko)) || !a.positions || !a.turn || !a.axis)
    return UMIC_ERR_INVALID_ARG;
  if ((a.qw == nullptr) != (a.kw == nullptr)) return UMIC_ERR_INVALID_ARG;
  if (a.D % 8 || a.D / 2 > kMaxHalf || a.Hq > (1 << 16) || a.Hk > (1 << 16))
    return UMIC_ERR_UNSUPPORTED;
  return UMIC_OK;
}

}  // namespace
}  // namespace umic
