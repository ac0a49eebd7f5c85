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
// workgroup takes a few tokens, forms their D/2 sines and cosines once in LDS,
// and shares them among all heads.
#include "common.hpp"

namespace umic {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;      // tokens of a workgroup
constexpr int kMaxHalf = 256;   // D/2 of the largest head

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
  SmallDiv group;   // lanes of a head row
  SmallDiv rows;    // head rows of a token
};

template <int VEC>
__device__ __forceinline__ void load_vec(const uint16_t* p, float* f) {
  if constexpr (VEC == 8)
    unpack8(ld_stream(reinterpret_cast<const u32x4*>(p)), f);
  else
    unpack4(*reinterpret_cast<const u32x2*>(p), f);
}

template <int VEC>
__device__ __forceinline__ void store_vec(uint16_t* p, const float* f) {
  if constexpr (VEC == 8)
    *reinterpret_cast<u32x4*>(p) = pack8(f);
  else
    *reinterpret_cast<u32x2*>(p) = pack4(f);
}

// A lane holds VEC elements of each half of a head row; `group` lanes (a power
// of two with the norm, whose sum runs over them; lanes past the row idle) hold
// a row.
template <int VEC, bool NORM>
__global__ __launch_bounds__(kThreads) void axial_kernel(AxialArgs a) {
  __shared__ float cs[kTokens][kMaxHalf][2];
  const int half = (int)a.D / 2;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const int here = (int)(a.T - t0 < kTokens ? a.T - t0 : kTokens);
  for (int i = threadIdx.x; i < here * half; i += kThreads) {
    const int t = i / half, f = i - t * half;
    const int ax = a.axis[f];
    float s = 0.0f, c = 1.0f;
    if (ax >= 0 && ax < a.A) {  // an axis that is not there does not turn
      const int64_t pos = a.positions[ax * a.p_sa + (t0 + t) * a.p_st];
      const int32_t frac = (int32_t)(((uint64_t)pos * a.turn[f]) >> 32);
      sincospif((float)frac * 0x1p-31f, &s, &c);
    }
    cs[t][f][0] = c * a.scale;
    cs[t][f][1] = s * a.scale;
  }
  __syncthreads();
  const int per = a.rows.d * a.group.d;  // lanes of a token
  const int chunks = half / VEC;
  for (int i = threadIdx.x; i < here * per; i += kThreads) {
    int c, h;
    const int row = div_small(a.group, i, c);
    const int t = div_small(a.rows, row, h);
    const int64_t tok = t0 + t;
    const bool active = c < chunks;
    const int kind = h < a.Hq ? 0 : h < a.Hq + a.Hk ? 1 : 2;
    const uint16_t* src;
    uint16_t* dst;
    bool write = active;
    if (kind == 0) {
      src = a.q + tok * a.q_st + h * a.q_sh;
      dst = a.qo + tok * a.qo_st + h * a.qo_sh;
    } else {
      const int hk = h - (int)a.Hq - (kind == 2 ? (int)a.Hk : 0);
      src = kind == 1 ? a.k + tok * a.k_st + hk * a.k_sh : a.v + tok * a.v_st + hk * a.v_sh;
      dst = kind == 1 ? a.ko : a.vo;
      if (a.slots) {  // a slot outside the pool is not written
        const int64_t slot = a.slots[tok];
        write = write && slot >= 0 && slot < a.slots_n;
        const int64_t page = slot >> a.shift, r = slot & (((int64_t)1 << a.shift) - 1);
        dst += page * a.ko_sb + hk * a.ko_sh + r * a.ko_st;
      } else {
        dst += tok * a.ko_st + hk * a.ko_sh;
      }
    }
    const int d = active ? c * VEC : 0;
    float lo[VEC], hi[VEC], ol[VEC], oh[VEC];
    load_vec<VEC>(src + d, lo);
    load_vec<VEC>(src + half + d, hi);
    if (kind == 2) {
      if (write) {
        store_vec<VEC>(dst + d, lo);
        store_vec<VEC>(dst + half + d, hi);
      }
      continue;
    }
    if constexpr (NORM) {
      float ss = 0.0f;
      if (active)
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss += lo[j] * lo[j] + hi[j] * hi[j];
      for (int m = 1; m < a.group.d; m <<= 1) ss += __shfl_xor(ss, m, kWave);
      const float r = rsqrt_cr(ss / (float)a.D + a.eps);
      const uint16_t* w = kind == 0 ? a.qw : a.kw;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        lo[j] = lo[j] * r * bf2f(w[d + j]);
        hi[j] = hi[j] * r * bf2f(w[half + d + j]);
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float co = cs[t][d + j][0], si = cs[t][d + j][1];
      ol[j] = lo[j] * co - hi[j] * si;
      oh[j] = hi[j] * co + lo[j] * si;
    }
    if (write) {
      store_vec<VEC>(dst + d, ol);
      store_vec<VEC>(dst + half + d, oh);
    }
  }
}

int launch_axial(AxialArgs& a, hipStream_t st) {
  const bool norm = a.qw != nullptr;
  int64_t low = a.q_st | a.q_sh | a.k_st | a.k_sh | a.qo_st | a.qo_sh | a.ko_st | a.ko_sh;
  uintptr_t ptr = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.qo | (uintptr_t)a.ko;
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
  const int64_t rows = a.Hq + a.Hk * (a.slots ? 2 : 1);
  if (group > kWave || rows * group * kTokens >= (1 << 22)) return UMIC_ERR_UNSUPPORTED;
  a.group = small_div((int)group);
  a.rows = small_div((int)rows);
  const int64_t blocks = (a.T + kTokens - 1) / kTokens;
  if (blocks > 0x7fffffff) return UMIC_ERR_UNSUPPORTED;
  auto* kern = vec == 8 ? (norm ? axial_kernel<8, true> : axial_kernel<8, false>)
                        : (norm ? axial_kernel<4, true> : axial_kernel<4, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
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
