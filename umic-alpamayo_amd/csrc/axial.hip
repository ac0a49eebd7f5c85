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
#include "axial.hpp"

namespace umic {
namespace {

template <int VEC, bool NORM, bool NT>
__global__ __launch_bounds__(kThreads) void axial_kernel(AxialArgs a) {
  extern __shared__ float cs[];
  axial_rows<VEC, NORM, NT>(a, blockIdx.x, cs);
}

int launch_axial(AxialArgs& a, hipStream_t st) {
  AxialShape s;
  if (const int e = axial_shape(a, s)) return e;
  const bool norm = a.qw != nullptr;
  auto* kern = s.vec == 4 ? (norm ? axial_kernel<4, true, false> : axial_kernel<4, false, false>)
               : s.lines  ? (norm ? axial_kernel<8, true, true> : axial_kernel<8, false, true>)
                          : (norm ? axial_kernel<8, true, false> : axial_kernel<8, false, false>);
  hipLaunchKernelGGL(kern, dim3(s.blocks), dim3(kThreads), s.lds, st, a);
  return launch_status();
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
