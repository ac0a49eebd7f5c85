// Attention of a request's new tokens over a paged cache of 8-bit codes, a scale for each
// block of 16 tokens and key head (codes.hpp):
//   o = sum_j p_j sv_j cv_j / sum_j p_j,  p_j = exp(scale sk_j q.ck_j - max).
//
// The kernels of attention.hip with half the bytes: codes become bf16 numbers, exactly,
// and the products, the softmax and the joins are theirs (attention.hpp).  A key tile of
// 16 is a block, so that its scales are a wave's scalars.
//
// Up to 16 rows: codes go from memory to registers; the scores of a tile are scaled by
// its key scale, its weights by its value scale.  More rows: codes are turned into scaled
// bf16 numbers once for the workgroup, on their way into LDS.
//
// A block whose scale is NaN reads as NaN: a row that sees one of its keys is NaN, others
// are as without it.
#include "attention.hpp"
#include "codes.hpp"

namespace umic {
namespace {

struct Attn8Args {
  AttnArgs a;  // first: args_again() reads it; its cache strides are in codes
  const float* ks;
  const float* vs;
  int64_t s_sb, s_sh;
};

__device__ __forceinline__ float scalar_f32(const float* p) {
  return *(const __attribute__((address_space(4))) float*)(uintptr_t)p;
}

__device__ __forceinline__ bool is_nan(float x) { return x != x; }

// Two tiles of 16 keys and their scales.
struct Place8 {
  Place p;
  float ks[2], vs[2];
};

__device__ __forceinline__ Place8 place8_of(const Attn8Args& x, const Keys& s, int h, int k0) {
  const Blocks blocks = blocks_of(x.a, s, k0);
  Place8 r;
  r.p = place_of(x.a, s, k0, blocks);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r.ks[i] = r.vs[i] = 0.0f;
    if (r.p.n[i]) {
      const int in = ((k0 + 16 * i) & ((1 << x.a.shift) - 1)) / kBlockTokens;
      const int64_t at = blocks.of[i] * x.s_sb + h * x.s_sh + in;
      r.ks[i] = scalar_f32(x.ks + at);
      r.vs[i] = scalar_f32(x.vs + at);
    }
  }
  return r;
}

// Rows that see a key of a tile whose values read as NaN (bit i of `wild`: tile i).
template <typename R>
__device__ __forceinline__ void spoil(R& r, int wild, int k0) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (wild >> i & 1)
#pragma unroll
      for (int nt = 0; nt < (int)(sizeof(r.lim) / sizeof(int)); ++nt)
        if (k0 + 16 * i < r.lim[nt])
#pragma unroll
          for (int e = 0; e < R::DV; ++e)
#pragma unroll
            for (int y = 0; y < 4; ++y) r.acc[nt][e][y] = __builtin_nanf("");
}

template <int D, int FORMAT>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attend8_few_kernel(Attn8Args x) {
  typedef Rows<D, 1, false> R;
  typedef Codes<FORMAT> C;
  constexpr int KK = R::KK, DV = R::DV;
  constexpr int KW = D / 16;  // words of a key's codes that a lane holds
  constexpr int VW = DV / 4;  // and of a value's
  constexpr int kTile = kStep * kWaves;
  __shared__ FewShared<D> lds;
  const AttnArgs& a = x.a;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;

  Scan scan = {};
  const int even = a.kv_len ? 0 : FewDeal::units(a.len);
  if (a.kv_len)
    scan = scan_units<FewDeal>(a, lds.sums);
  else
    scan.all = even * a.B;
  const FewDeal deal((unsigned)(scan.all * a.Hk), a.nwg, a.some);
  const int wg = dealt_wg(deal.nwg);
  if (wg >= 0) {
    Walk<FewDeal, false> walk;
    walk.start(a, deal, scan, even, wg, lds.found);
    R r;
    Segment seg, nxt;
    int split = 0;
    Place8 here;
    u32x4 kc[2][KW / 4];
    uint32_t vc[8][VW];
    // a lane's 16 codes of a key at a time, those of two steps of the product
    auto load_k = [&](const Place& p) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* kp = (const uint8_t*)a.k + p.at[i];
        const unsigned off = __umul24(min(n16, max(p.n[i] - 1, 0)), a.c_ss) + g4 * 16;
#pragma unroll
        for (int w = 0; w < KW / 4; ++w)
          kc[i][w] = ld_stream(reinterpret_cast<const u32x4*>(kp + off + w * 64));
      }
    };
    auto load_v = [&](const Place& p) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2;
        const unsigned off =
            __umul24(min(4 * g4 + (j & 3), max(p.n[i] - 1, 0)), a.c_ss) + n16 * DV;
        const uint32_t* vp = reinterpret_cast<const uint32_t*>((const uint8_t*)a.v + p.at[i] + off);
#pragma unroll
        for (int w = 0; w < VW; ++w) vc[j][w] = vp[w];
      }
    };
    auto first_of = [&](const Segment& s) {
      return place8_of(x, keys_of(a, s), s.h, s.t0 * kTile + wave * kStep);
    };
    walk.next(a, seg);  // a dealt workgroup has one
    here = first_of(seg);
    load_k(here.p);
    load_v(here.p);
    r.template load_q<true>(a, seg, 0, n16, g4);
    for (bool go = true; go;) {
      go = walk.next(a, nxt);
      const Place8 turn = go ? first_of(nxt) : here;
      bool turned = false;  // the next segment's keys are on their way
      const Keys keys = keys_of(a, seg);
      r.clear();
      for (int t = seg.t0; t < seg.t1; ++t) {
        const int k0 = t * kTile + wave * kStep, k1 = k0 + kTile;
        if (k0 >= r.hi) break;
        const bool more = t + 1 < seg.t1 && k1 < r.hi;
        Place8 next = turn;
        if (more) next = place8_of(x, keys, seg.h, k1);
        turned = !more;
        f32x4_t sc[1][2] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            const u32x2 lo = C::four(kc[i][kk / 2][kk % 2 * 2]);
            const u32x2 hi = C::four(kc[i][kk / 2][kk % 2 * 2 + 1]);
            sc[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                as_bf(u32x4{lo[0], lo[1], hi[0], hi[1]}), as_bf(r.q[0][kk]), sc[0][i], 0, 0, 0);
          }
          sc[0][i] *= here.ks[i];
        }
        if (more || go) load_k(next.p);  // under the softmax and the second product
        if (k0 + kStep > r.lo || here.p.n[0] < 16 || here.p.n[1] < 16) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int at = 4 * g4 + (j & 3), key = k0 + 16 * (j >> 2) + at;
            const bool there = at < here.p.n[j >> 2];
            if (!there || key >= r.lim[0]) sc[0][j >> 2][j & 3] = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < VW; ++w) vc[j][w] = there ? vc[j][w] : 0;
          }
        }
        float vs[2] = {here.vs[0], here.vs[1]};
        const int wild = (is_nan(vs[0]) ? 1 : 0) | (is_nan(vs[1]) ? 2 : 0);
        if (wild) {
          spoil(r, wild, k0);
          if (wild & 1) vs[0] = 0.0f;
          if (wild & 2) vs[1] = 0.0f;
        }
        u32x4 ph[1], pl[1];
        r.template weights<true>(sc, a.c, ph, pl, vs);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t o[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) C::turn(vc[2 * j][w], vc[2 * j + 1][w], o[j]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bf16x8_t v = as_bf(u32x4{o[0][c], o[1][c], o[2][c], o[3][c]});
            f32x4_t& to = r.acc[0][4 * w + c];
            to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, as_bf(ph[0]), to, 0, 0, 0);
            to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, as_bf(pl[0]), to, 0, 0, 0);
          }
        }
        if (more || go) load_v(next.p);
        here = next;
      }
      if (go) {
        if (!turned) {
          load_k(turn.p);
          load_v(turn.p);
        }
        here = turn;
        r.template load_q<true>(a, nxt, 0, n16, g4);
      }
      join_waves<D, false>(args_again(), r, seg, lds, wg, split);
      seg = nxt;
    }
    join_parts<D>(args_again(), deal, lds, split);
  }
  const AttnArgs z = args_again();
  if (z.counters) zero_rows<D>(z);
}

// More rows: each wave has 16 NT of the workgroup's 64 NT.  Codes are asked for two steps
// of 32 keys ahead, in registers, and go scaled into one of two buffers of LDS while the
// other is read.  Chunks of a row are permuted as attention.hip's.
template <int D, int NT, int FORMAT>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void attend8_many_kernel(Attn8Args x) {
  typedef Rows<D, NT, true> R;
  typedef Codes<FORMAT> C;
  constexpr int KK = R::KK, DV = R::DV;
  constexpr int CH = D / 8;                  // 16-byte chunks of a row in LDS
  constexpr int PT = D / 32;                 // words of codes a thread moves of K (and V)
  constexpr int kBlock = 16 * NT * kWaves;   // rows of a workgroup
  __shared__ int sums[kWaves];
  __shared__ int found[2];
  __shared__ u32x4 kv[2][2][kStep * CH];     // [buffer][K, V]
  __shared__ int wilds[2][2];                // [buffer][tile]: its values read as NaN
  const AttnArgs& a = x.a;
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
  // eight threads to a key, a wave's keys of one tile
  const int row = threadIdx.x >> 3, part = threadIdx.x & 7, tile = wave >> 1;
  struct Raw {
    uint32_t k[PT], v[PT];
    float ks, vs;
  } raw[2];
  while (walk.next(a, seg)) {
    const int r0 = seg.rb * kBlock + wave * 16 * NT;
    int end = seg.len;  // the block's last key that any row sees
    if (a.causal)
      end = min(end, seg.len - seg.fresh + quot(min((seg.rb + 1) * kBlock, rows) - 1, a.G) + 1);
    const int t1 = min(seg.t1, (max(end, 0) + kStep - 1) / kStep);
    const Keys keys = keys_of(a, seg);
    auto load = [&](int t, Raw& w) {
      const Place8 p = place8_of(x, keys, seg.h, t * kStep);
      const int n = tile ? p.p.n[1] : p.p.n[0];
      const int64_t at = (tile ? p.p.at[1] : p.p.at[0]) +
                         __umul24(min(row & 15, max(n - 1, 0)), a.c_ss) + part * (PT * 4);
      w.ks = tile ? p.ks[1] : p.ks[0];
      w.vs = tile ? p.vs[1] : p.vs[0];
      const uint32_t* kp = reinterpret_cast<const uint32_t*>((const uint8_t*)a.k + at);
      const uint32_t* vp = reinterpret_cast<const uint32_t*>((const uint8_t*)a.v + at);
#pragma unroll
      for (int i = 0; i < PT; ++i) w.k[i] = kp[i], w.v[i] = vp[i];
    };
    auto store = [&](int t, const Raw& w) {
      const int buf = t & 1;
      const bool wild = is_nan(w.vs);
      const float vs = wild ? 0.0f : w.vs;
#pragma unroll
      for (int c = 0; c < PT / 2; ++c) {
        const int chunk = part * (PT / 2) + c;
        const u32x2 k0 = C::four(w.k[2 * c], w.ks), k1 = C::four(w.k[2 * c + 1], w.ks);
        const u32x2 v0 = C::four(w.v[2 * c], vs), v1 = C::four(w.v[2 * c + 1], vs);
        kv[buf][0][row * CH + (chunk ^ k_swizzle(row & 15))] = u32x4{k0[0], k0[1], k1[0], k1[1]};
        kv[buf][1][row * CH + (chunk ^ v_swizzle(row))] = u32x4{v0[0], v0[1], v1[0], v1[1]};
      }
      if ((wave & 1) == 0 && lane == 0) wilds[buf][tile] = wild;
    };
    __syncthreads();  // the last segment's reads are done
    if (seg.t0 < t1) load(seg.t0, raw[0]);
    if (seg.t0 + 1 < t1) load(seg.t0 + 1, raw[1]);
    r.load_q(a, seg, r0, n16, g4);
    r.clear();
    if (seg.t0 < t1) {
      store(seg.t0, raw[0]);
      if (seg.t0 + 2 < t1) load(seg.t0 + 2, raw[0]);
    }
    auto step = [&](int t, Raw& next) {
      const int k0 = t * kStep;
      __syncthreads();  // this step's keys are there, those of the step before have been read
      if (t + 1 < t1) {
        store(t + 1, next);
        if (t + 3 < t1) load(t + 3, next);
      }
      if (k0 >= r.hi || r0 >= rows) return;
      const u32x4* const ks = kv[t & 1][0];
      const u32x4* const vs = kv[t & 1][1];
      u32x4 kf[2][KK];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kf[i][kk] = ks[(16 * i + n16) * CH + ((kk * 4 + g4) ^ k_swizzle(n16))];
      f32x4_t sc[NT][2];
      r.scores(kf, sc);
      // as in attention.hip: 4 keys by 16 columns turned over 16 lanes
      uint32_t vr[R::VR];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = 16 * i + 4 * g4 + (n16 >> 2);
#pragma unroll
        for (int e = 0; e < DV; ++e) {
          const u32x4* const c = vs + at * CH + ((2 * e + ((n16 >> 1) & 1)) ^ v_swizzle(at));
          const uint64_t w = __builtin_bit_cast(
              uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_s16x4*)(reinterpret_cast<const uint64_t*>(c) + (n16 & 1))));
          vr[4 * e + 2 * i] = (uint32_t)w;
          vr[4 * e + 2 * i + 1] = (uint32_t)(w >> 32);
        }
      }
      const Place here = place_of(a, keys, k0, blocks_of(a, keys, k0));
      if (k0 + kStep > r.lo || here.n[0] < 16 || here.n[1] < 16) r.mask(sc, vr, here.n, k0, g4);
      const int wild = uniform(wilds[t & 1][0]) | uniform(wilds[t & 1][1]) << 1;
      if (wild) spoil(r, wild, k0);
      u32x4 ph[NT], pl[NT];
      r.weights(sc, a.c, ph, pl);
      r.product(vr, ph, pl);
    };
    for (int t = seg.t0; t < t1; t += 2) {
      step(t, raw[1]);
      if (t + 1 < t1) step(t + 1, raw[0]);
    }
    const AttnArgs args = args_again();
    const int slot = wg * 2 + (seg.t0 == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum = r.l[nt];
      sum += __shfl_xor(sum, 16, kWave);
      sum += __shfl_xor(sum, 32, kWave);
      const int at = r0 + nt * 16 + n16;
      const bool padded = quot(at, args.G) >= seg.fresh;
      if (at < rows) write_rows<D, NT>(args, seg, r, nt, at, slot, padded, sum);
    }
  }
}

template <int D, int NT, int FORMAT>
int launch8_many(const Attn8Args& x, hipStream_t st) {
  const dim3 grid((unsigned)((x.a.nwg + 7) / 8 * 8)), threads(kThreads);
  hipLaunchKernelGGL((attend8_many_kernel<D, NT, FORMAT>), grid, threads, 0, st, x);
  if (const int e = launch_status()) return e;
  return launch_join_many<D, NT>(x.a, st);
}

template <int D, int FORMAT>
int launch8(const Shape& s, const Attn8Args& x, hipStream_t st) {
  if constexpr (D <= 128)
    if (s.nt == 2) return launch8_many<D, 2, FORMAT>(x, st);
  if (s.nt) return launch8_many<D, 1, FORMAT>(x, st);
  const dim3 grid((unsigned)((x.a.nwg + 7) / 8 * 8)), threads(kThreads);
  hipLaunchKernelGGL((attend8_few_kernel<D, FORMAT>), grid, threads, 0, st, x);
  const int e = launch_status();
  if (e || x.a.counters) return e;
  return launch_join_few<D>(x.a, st);
}

}  // namespace
}  // namespace umic

extern "C" int umic_cache8_attention_bf16(
    const umic_cache8_t* cache, const void* q, void* out, const int32_t* table,
    const int32_t* kv_lens, const int32_t* q_lens, int64_t B, int64_t S, int64_t Hq, int64_t q_sb,
    int64_t q_ss, int64_t q_sh, int64_t o_sb, int64_t o_ss, int64_t o_sh, int64_t table_ld,
    int64_t table_w, int64_t kv_len, int causal, float scale, int32_t* counters, void* workspace,
    int64_t workspace_bytes, void* stream) {
  using namespace umic;
  int64_t cap;
  if (const int e = check_cache8(cache, cap, table_w)) return e;
  const umic_cache8_t& c = *cache;
  const int64_t D = c.head_dim;
  const AttnCall call = {q,      c.k_codes, c.v_codes, out,  table, kv_lens, q_lens, B,    S,
                         Hq,     c.heads,   D,         q_sb, q_ss,  q_sh,    o_sb,   o_ss, o_sh,
                         c.c_sb, c.c_sh,    c.c_ss,    c.pages, c.page_size, table_ld, table_w,
                         kv_len, causal,    scale,     counters, workspace, workspace_bytes};
  Attn8Args x = {};
  Shape s;
  if (!table && B > 0 && S > 0 && Hq > 0) return UMIC_ERR_INVALID_ARG;
  if (const int e = attn_args(call, 16, x.a, s)) return e == 1 ? UMIC_OK : e;
  x.ks = c.k_scale, x.vs = c.v_scale, x.s_sb = c.s_sb, x.s_sh = c.s_sh;
  hipStream_t st = as_stream(stream);
  const bool f = c.format == UMIC_CODES_INT8;
  if (D == 64)
    return f ? launch8<64, UMIC_CODES_INT8>(s, x, st) : launch8<64, UMIC_CODES_E4M3>(s, x, st);
  if (D == 128)
    return f ? launch8<128, UMIC_CODES_INT8>(s, x, st) : launch8<128, UMIC_CODES_E4M3>(s, x, st);
  return f ? launch8<256, UMIC_CODES_INT8>(s, x, st) : launch8<256, UMIC_CODES_E4M3>(s, x, st);
}
