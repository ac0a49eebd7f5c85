// Rotary positions of several axes (time, height, width of images and video),
// from the positions themselves, with the per-head RMSNorm in front and the
// paged cache behind.
//
// Pair f of a head row, elements f and f + D/2, turns by positions[axis[f]][t] *
// inv_freq[f]:   x_f cos - x_{f+D/2} sin,   x_{f+D/2} cos + x_f sin.
// The angle is kept as a fraction of a turn in 64-bit fixed point: turn[f] =
// round(2^64 inv_freq[f] / 2 pi), and position * turn[f] modulo 2^64 is the
// angle's fraction whatever the position, to |position| 2^-65 of a turn.  (In
// fp32 the product of a position near 2^20 and a frequency near 1 is off by
// 2^-4 rad.)  Everything else is fp32, rounded once to bf16.
//
// HBM-bound at prompt sizes: each row is read once and written once.  A
// workgroup takes a few tokens: its threads' first loads are on their way while
// the tokens' D/2 sines and cosines are formed, once for all heads, in LDS.  32 + 8
// heads of 128 into the pages: 16381 tokens 67 us, at the copy of their bytes (5.9
// TB/s); 3100 with the norm 16.8, 12% over it; 8 tokens 5.2.
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

// A lane holds VEC elements of each half of a head row; `group` lanes (a power
// of two with the norm, whose sum runs over them; lanes past the row idle) hold
// a row.  NT: stores past the caches, where the halves of a row are whole lines
// (16381 tokens of 32 + 8 heads of 128: 72 us for 80; rows of 80, which are not,
// 46 for 40).
template <int VEC, bool NORM, bool NT>
__global__ __launch_bounds__(kThreads) void axial_kernel(AxialArgs a) {
  constexpr int kItems = kItemsOf<NORM>;
  extern __shared__ float cs[];  // [token][pair] (cos, sin)
  const int half = a.half.d;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
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
      at[u] = t * half + d;
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
      const int32_t frac = (int32_t)(((uint64_t)pos * a.turn[f]) >> 32);
      sincospif((float)frac * 0x1p-31f, &s, &c);
    }
    cs[2 * i] = c * a.scale;
    cs[2 * i + 1] = s * a.scale;
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
        const float co = cs[2 * (t + j)], si = cs[2 * (t + j) + 1];
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

int launch_axial(AxialArgs& a, hipStream_t st) {
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
  const bool lines = half % 64 == 0;
  auto* kern = vec == 4 ? (norm ? axial_kernel<4, true, false> : axial_kernel<4, false, false>)
               : lines  ? (norm ? axial_kernel<8, true, true> : axial_kernel<8, false, true>)
                        : (norm ? axial_kernel<8, true, false> : axial_kernel<8, false, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads),
                     (size_t)a.tokens * half * 2 * sizeof(float), st, a);
  return launch_status();
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

extern "C" int umic_axial_rope_bf16(const void* q, const void* k, void* q_out, void* k_out,
                                    const int64_t* positions, const uint64_t* turn,
                                    const int32_t* axis, float scale, const void* q_w,
                                    const void* k_w, float eps, int64_t T, int64_t Hq, int64_t Hk,
                                    int64_t D, int64_t axes, int64_t p_sa, int64_t p_st,
                                    int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                                    int64_t qo_st, int64_t qo_sh, int64_t ko_st, int64_t ko_sh,
                                    void* stream) {
  using namespace umic;
  AxialArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k;
  a.qo = (uint16_t*)q_out, a.ko = (uint16_t*)k_out;
  a.positions = positions, a.turn = turn, a.axis = axis;
  a.qw = (const uint16_t*)q_w, a.kw = (const uint16_t*)k_w;
  a.T = T, a.Hq = Hq, a.Hk = Hk, a.D = D, a.A = axes, a.p_sa = p_sa, a.p_st = p_st;
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh;
  a.qo_st = qo_st, a.qo_sh = qo_sh, a.ko_st = ko_st, a.ko_sh = ko_sh;
  a.eps = eps, a.scale = scale;
  if (int e = check_axial(a)) return e < 0 ? e : UMIC_OK;
  return launch_axial(a, as_stream(stream));
}

extern "C" int umic_axial_rope_append_bf16(
    const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages,
    const int64_t* positions, const uint64_t* turn, const int32_t* axis, const int64_t* slots,
    float scale, const void* q_w, const void* k_w, float eps, int64_t T, int64_t Hq, int64_t Hk,
    int64_t D, int64_t axes, int64_t p_sa, int64_t p_st, int64_t q_st, int64_t q_sh, int64_t k_st,
    int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t qo_st, int64_t qo_sh, int64_t c_sb,
    int64_t c_sh, int64_t c_ss, int64_t pages, int64_t page_size, void* stream) {
  using namespace umic;
  AxialArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.qo = (uint16_t*)q_out, a.ko = (uint16_t*)k_pages, a.vo = (uint16_t*)v_pages;
  a.positions = positions, a.turn = turn, a.axis = axis, a.slots = slots;
  a.qw = (const uint16_t*)q_w, a.kw = (const uint16_t*)k_w;
  a.T = T, a.Hq = Hq, a.Hk = Hk, a.D = D, a.A = axes, a.p_sa = p_sa, a.p_st = p_st;
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  a.qo_st = qo_st, a.qo_sh = qo_sh, a.ko_sb = c_sb, a.ko_sh = c_sh, a.ko_st = c_ss;
  a.eps = eps, a.scale = scale;
  if (pages < 0 || page_size <= 0) return UMIC_ERR_INVALID_ARG;
  if (int e = check_axial(a)) return e < 0 ? e : UMIC_OK;
  if (!slots || (Hk && (!v || !v_pages))) return UMIC_ERR_INVALID_ARG;
  if (page_size < 16 || (page_size & (page_size - 1)) || page_size > ((int64_t)1 << 30) ||
      pages > ((int64_t)1 << 30))
    return UMIC_ERR_UNSUPPORTED;
  a.shift = __builtin_ctzll((unsigned long long)page_size);
  a.slots_n = pages * page_size;
  return launch_axial(a, as_stream(stream));
}
