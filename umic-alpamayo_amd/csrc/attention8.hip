// Attention of a request's new tokens over a paged cache of 8-bit codes, a scale for each
// block of 16 tokens and key head (codes.hpp):
//   o = sum_j p_j sv_j cv_j / sum_j p_j,  p_j = exp(scale sk_j q.ck_j - max).
//
// The kernels of attention.hip with half the bytes: codes become bf16 numbers, exactly,
// and the products, the softmax and the joins are theirs (attention.hpp).  A key tile of
// 16 is a block, so that its scales are a wave's scalars.
//
// Up to 16 rows: codes go from memory to registers; the scores of a tile are scaled by
// its key scale, its weights by its value scale.  Where a scale or an element of q is 2^97
// or more, that can pass what fp32 holds: such a part of a segment is done again, from
// scaled codes.  More rows: codes are turned into scaled bf16 numbers once for the
// workgroup, on their way into LDS.
//
// A block whose scale is NaN reads as NaN: a row that sees one of its keys is NaN, others
// are as without it.
#include <type_traits>

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

__device__ __forceinline__ Attn8Args args8_again() {
  typedef const __attribute__((address_space(4))) Attn8Args* Args;
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Attn8Args*)p;
}

__device__ __forceinline__ float scalar_f32(const float* p) {
  return *(const __attribute__((address_space(4))) float*)(uintptr_t)p;
}

__device__ __forceinline__ bool is_nan(float x) { return x != x; }

// A segment's codes and scales, of its key head; row j is row j % 2^shift of page
// row[j >> shift].
struct View {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* row;
  int len;
};

__device__ __forceinline__ View view_of(const Attn8Args& x, const Segment& s) {
  View w;
  const int64_t codes = s.h * x.a.c_sh, scales = s.h * x.s_sh;
  w.k = (const uint8_t*)x.a.k + codes;
  w.v = (const uint8_t*)x.a.v + codes;
  w.ks = x.ks + scales;
  w.vs = x.vs + scales;
  w.row = x.a.table + s.b * x.a.table_ld;
  w.len = s.len;
  return w;
}

// A tile of 16 keys: where it lies, the first n rows of it there, and its scales.
struct Tile {
  int64_t at;
  int n;
  float ks, vs;
};

__device__ __forceinline__ Tile tile_of(const Attn8Args& x, const View& w, int key) {
  Tile r;
  const int in = key & ((1 << x.a.shift) - 1);
  const unsigned page =
      (unsigned)scalar_i32(w.row + min(key >> x.a.shift, (w.len - 1) >> x.a.shift));
  const bool out = page >= (unsigned)x.a.blocks;  // of the pool: not there
  r.n = out ? 0 : min(max(w.len - key, 0), 16);
  // rows and scales of a tile that is not there are others': nothing of it counts
  const int64_t p = out ? 0 : page;
  r.at = p * x.a.c_sb + (int64_t)in * x.a.c_ss;
  const int64_t block = p * x.s_sb + in / kBlockTokens;
  r.ks = scalar_f32(w.ks + block);
  r.vs = scalar_f32(w.vs + block);
  return r;
}

// Rows that see a key of a tile whose values read as NaN (bit i of `wild`, of two: tile i): their
// sum makes all of their output NaN.
template <typename R>
__device__ __forceinline__ void spoil(R& r, int wild, int k0) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (wild >> i & 1)
#pragma unroll
      for (int nt = 0; nt < (int)(sizeof(r.lim) / sizeof(int)); ++nt)
        if (k0 + 16 * i < r.lim[nt]) r.l[nt] = __builtin_nanf("");
}

// Four codes as scaled bf16 numbers, infinite ones as the largest.
template <typename C>
__device__ __forceinline__ u32x2 scaled4(uint32_t w, float scale) {
  const u32x2 v = C::four(w, scale);
  return C::kPasses ? at_most(v) : v;
}

// The larger one's bits: numbers above 0, and NaN above all.
__device__ __forceinline__ int top_of(float a, float b) {
  return max((int)__float_as_uint(a), (int)__float_as_uint(b));
}
// Of a tile that is there: a block that no token has come to can have any scale.
__device__ __forceinline__ int top_of(const Tile& p) { return p.n ? top_of(p.ks, p.vs) : 0; }

// attention.hpp's Deal with the remainder spread evenly, workgroup w beginning at w all /
// nwg: where the workgroups of a segment come out even, none has parts of two (a request
// of 40000 keys 23.6 us for 27.7, four of 12000 22.9 for 26.6).  If the chip's workgroups
// have less than LEAST units each, no more than `some`, of EACH or more.
template <int TILE, int LEAD, int LEAST, int EACH>
struct EvenDeal {
  unsigned all, each, more;
  int nwg;

  static __device__ __forceinline__ int tiles(int keys) { return (keys + TILE - 1) / TILE; }
  static __device__ __forceinline__ int units(int keys) {
    return keys > 0 ? tiles(keys) + LEAD : 0;
  }
  __device__ __forceinline__ EvenDeal(unsigned all, int most, int some) : all(all) {
    nwg = all / LEAST >= (unsigned)most ? most : min((int)((all + EACH - 1) / EACH), some);
    each = nwg ? all / (unsigned)nwg : 0;
    more = all - each * (unsigned)nwg;
  }
  __device__ __forceinline__ int begin(unsigned wg) const {
    return (int)(wg * each + wg * more / (unsigned)nwg);
  }
  __device__ __forceinline__ int holder(unsigned unit) const {
    // to one workgroup: there are 4096 at most, and the three roundings are of 2^-24 each
    int w = min((int)((float)unit * ((float)nwg / (float)all)), nwg - 1);
    if ((unsigned)begin(w) > unit) --w;
    if ((unsigned)begin(w + 1) <= unit) ++w;
    return w;
  }
  __device__ __forceinline__ void holders(unsigned at, int tiles, int& w0, int& w1) const {
    w0 = holder(at + LEAD);
    w1 = holder(at + LEAD + tiles - 1);
  }
};

// Single tokens: 128 keys; a segment's start and end cost some two of them (64 ragged
// requests 32 us; counted as nothing 39, as one or three 32 and 33).  EACH: two units, as a
// part costs its join too (one token over 9000 keys of two heads, 16 rows each, 20 us for
// 26; over 3100 of eight 11.9 either way; of three units 12.1).
typedef EvenDeal<kStep * kWaves, 2, 5, 2> Few8Deal;

// Workgroups of a CU.  (Three: 64 ragged requests 31 us for 32, 128 requests of 3000 keys
// 148 for 132, two of 131001 98 for 94.  One: 57, 161, 110.)
constexpr int few8_of(int64_t D) { return D <= 128 ? 2 : 1; }

// Up to 16 rows: attention.hip's kernel, a wave to 32 of a tile's 128 keys, the loads of a
// step in flight while the one before is computed.
// What bounds it: HBM where the keys are many (64 requests of 8000 keys 170 us, 6.2 TB/s);
// a request of 3100 keys 10.5 us (bf16 rows 10.2 beside it; 10 to 14 from one process to
// another), of which 4 pass until its first keys are there and 3 to join; of a step's 350
// vector instructions int8 codes take 192 (one to a number, half one to pair it) and e4m3's
// 80.
template <int D, int FORMAT>
__global__ __launch_bounds__(kThreads, few8_of(D)) void attend8_few_kernel(Attn8Args x) {
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
  const int even = a.kv_len ? 0 : Few8Deal::units(a.len);
  if (a.kv_len)
    scan = scan_units<Few8Deal>(a, lds.sums);
  else
    scan.all = even * a.B;
  const Few8Deal deal((unsigned)(scan.all * a.Hk), a.nwg, a.some);
  const int wg = dealt_wg(deal.nwg);
  if (wg >= 0) {
    Walk<Few8Deal, false> walk;
    walk.start(a, deal, scan, even, wg, lds.found);
    R r;
    Segment seg, nxt;
    int split = 0;
    Tile here[2];
    u32x4 kc[2][KW / 4];
    uint32_t vc[8][VW];
    // a lane's 16 codes of a key at a time, those of two steps of the product
    auto load_k = [&](const uint8_t* k, const Tile (&p)[2], int c_ss) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* kp = k + p[i].at;
        const unsigned off = __umul24(min(n16, max(p[i].n - 1, 0)), c_ss) + g4 * 16;
#pragma unroll
        for (int j = 0; j < KW / 4; ++j)
          kc[i][j] = ld_stream(reinterpret_cast<const u32x4*>(kp + off + j * 64));
      }
    };
    auto load_v = [&](const uint8_t* v, const Tile (&p)[2], int c_ss) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2;
        const unsigned off = __umul24(min(4 * g4 + (j & 3), max(p[i].n - 1, 0)), c_ss) + n16 * DV;
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(v + p[i].at + off);
#pragma unroll
        for (int c = 0; c < VW; ++c) vc[j][c] = vp[c];
      }
    };
    // Keys that are not there, and those that a row does not see.
    auto mask = [&](f32x4_t (&sc)[1][2], const Tile (&p)[2], int k0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = 4 * g4 + (j & 3), key = k0 + 16 * (j >> 2) + at;
        const bool there = at < p[j >> 2].n;
        if (!there || key >= r.lim[0]) sc[0][j >> 2][j & 3] = -__builtin_inff();
#pragma unroll
        for (int c = 0; c < VW; ++c) vc[j][c] = there ? vc[j][c] : 0;
      }
    };
    auto tiles = [](const Attn8Args& x, const View& w, int k0, Tile (&p)[2]) {
      p[0] = tile_of(x, w, k0);
      p[1] = tile_of(x, w, k0 + 16);
    };
    // A segment's tiles of this wave from scaled codes, one step at a time.
    auto again = [&](const Segment& s, const View& w) {
      const Attn8Args y = args8_again();
      r.clear();
#pragma unroll 1
      for (int t = s.t0; t < s.t1; ++t) {
        const int k0 = t * kTile + wave * kStep;
        Tile p[2];
        tiles(y, w, k0, p);
        load_k(w.k, p, y.a.c_ss);
        load_v(w.v, p, y.a.c_ss);
        f32x4_t sc[1][2] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            const u32x2 lo = scaled4<C>(kc[i][kk / 2][kk % 2 * 2], p[i].ks);
            const u32x2 hi = scaled4<C>(kc[i][kk / 2][kk % 2 * 2 + 1], p[i].ks);
            sc[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                as_bf(u32x4{lo[0], lo[1], hi[0], hi[1]}), as_bf(r.q[0][kk]), sc[0][i], 0, 0, 0);
          }
        mask(sc, p, k0);
        u32x4 ph[1], pl[1];
        r.weights(sc, y.a.c, ph, pl);
        float vs[2];
        int wild = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          vs[i] = p[i].n ? p[i].vs : 0.0f;
          if (is_nan(vs[i])) wild |= 1 << i, vs[i] = 0.0f;
        }
        uint32_t v[R::VR];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            const u32x2 x = scaled4<C>(vc[j][c], vs[j >> 2]);
            v[R::VW * j + 2 * c] = x[0], v[R::VW * j + 2 * c + 1] = x[1];
          }
        r.product(v, ph, pl);
        if (wild) spoil(r, wild, k0);
      }
    };
    bool go = walk.next(a, seg);  // not where a segment's start is all that it was dealt
    View view, after;
    if (go) {
      view = view_of(x, seg);
      tiles(x, view, seg.t0 * kTile + wave * kStep, here);
      load_k(view.k, here, a.c_ss);
      load_v(view.v, here, a.c_ss);
      r.template load_q<true>(a, seg, 0, n16, g4);
    }
    while (go) {
      const Attn8Args y = args8_again();
      go = walk.next(y.a, nxt);
      Tile turn[2] = {here[0], here[1]};
      after = view;
      if (go) {
        after = view_of(y, nxt);
        tiles(y, after, nxt.t0 * kTile + wave * kStep, turn);
      }
      bool turned = false;  // the next segment's keys are on their way
      int top = 0;          // bits of the largest scale
      r.clear();
      for (int t = seg.t0; t < seg.t1; ++t) {
        const int k0 = t * kTile + wave * kStep, k1 = k0 + kTile;
        if (k0 >= r.hi) break;
        const bool more = t + 1 < seg.t1 && k1 < r.hi;
        Tile next[2] = {turn[0], turn[1]};
        if (more) tiles(y, view, k1, next);
        const uint8_t* const from_k = more ? view.k : after.k;
        const uint8_t* const from_v = more ? view.v : after.v;
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
          sc[0][i] *= here[i].ks;
        }
        if (more || go) load_k(from_k, next, y.a.c_ss);  // under the softmax and the second product
        if (k0 + kStep > r.lo || here[0].n < 16 || here[1].n < 16) {
          mask(sc, here, k0);
        }
        float vs[2] = {here[0].n ? here[0].vs : 0.0f, here[1].n ? here[1].vs : 0.0f};
        const int wild = (is_nan(vs[0]) ? 1 : 0) | (is_nan(vs[1]) ? 2 : 0);
        if (wild & 1) vs[0] = 0.0f;
        if (wild & 2) vs[1] = 0.0f;
        top = max(top, max(top_of(here[0]), top_of(here[1])));
        u32x4 ph[1], pl[1];
        r.template weights<true>(sc, y.a.c, ph, pl, vs);
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
        if (wild) spoil(r, wild, k0);
        if (more || go) load_v(from_v, next, y.a.c_ss);
        here[0] = next[0], here[1] = next[1];
      }
      // q is looked at here: ahead of the loop its wait changed those inside (a token over
      // 131001 keys 97 us for 93)
      uint32_t any = 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) any |= wide_q(r.q[0][kk]);
      if (__builtin_expect(top >= kWideBits || __any(any != 0), 0)) {
        turned = false;
        again(seg, view);
      }
      if (go) {
        const AttnArgs z = args_again();
        if (!turned) {
          load_k(after.k, turn, z.c_ss);
          load_v(after.v, turn, z.c_ss);
        }
        here[0] = turn[0], here[1] = turn[1];
        view = after;
        r.template load_q<true>(z, nxt, 0, n16, g4);
      }
      join_waves<D, false>(args_again(), r, seg, lds, wg, split);
      seg = nxt;
    }
    join_parts<D>(args_again(), deal, lds, split);
  }
  const AttnArgs z = args_again();
  if (z.counters) zero_rows<D>(z);
}

// More rows: each wave has 16 NT of the workgroup's 64 NT.  Codes are asked for a step of
// 32 keys ahead, in registers, and go scaled into one of two buffers of LDS while the
// other is read.  Two steps are written out, so that the buffers' addresses are known (128
// tokens over 65536 keys 216 us for 246).  Chunks of a row are permuted as attention.hip's.
// What bounds it: attention.hip's matrix and vector instructions, and 16 (e4m3) or 80
// (int8) vector ones of a wave's step for the codes: 128 tokens over 65536 keys 216 and 235
// us (640 and 580 TFLOP/s; bf16 rows 233), four 128-token chunks 47 and 48 (47), of which
// the joins take 13; 32 tokens over 3126 keys 18 (18).  (Codes asked for two steps ahead:
// the same, and 6% slower through LDS.)
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
  __shared__ int marks[2][2];  // [buffer][tile] 1: its values read as NaN, 4: not all is there
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
  uint32_t raw_k[PT], raw_v[PT];
  float raw_ks, raw_vs;
  bool raw_out;
  while (walk.next(args_again(), seg)) {
    const Attn8Args y = args8_again();
    const int r0 = seg.rb * kBlock + wave * 16 * NT;
    int end = seg.len;  // the block's last key that any row sees
    if (y.a.causal)
      end = min(end, seg.len - seg.fresh + quot(min((seg.rb + 1) * kBlock, rows) - 1, y.a.G) + 1);
    const int t1 = min(seg.t1, (max(end, 0) + kStep - 1) / kStep);
    const View view = view_of(y, seg);
    auto load = [&](int t) {
      const Tile p = tile_of(y, view, t * kStep + 16 * tile);
      const unsigned off = __umul24(min(row & 15, max(p.n - 1, 0)), y.a.c_ss) + part * (PT * 4);
      raw_ks = p.ks;
      raw_vs = p.n ? p.vs : 0.0f;
      raw_out = p.n < 16;
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(view.k + p.at + off);
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(view.v + p.at + off);
#pragma unroll
      for (int i = 0; i < PT; ++i) raw_k[i] = kp[i], raw_v[i] = vp[i];
    };
    auto store = [&](auto buffer) {
      constexpr int buf = buffer;
      const bool wild = is_nan(raw_vs);
      const float vs = wild ? 0.0f : raw_vs;
#pragma unroll
      for (int c = 0; c < PT / 2; ++c) {
        const int chunk = part * (PT / 2) + c;
        const u32x2 k0 = C::four(raw_k[2 * c], raw_ks), k1 = C::four(raw_k[2 * c + 1], raw_ks);
        const u32x2 v0 = C::four(raw_v[2 * c], vs), v1 = C::four(raw_v[2 * c + 1], vs);
        kv[buf][0][row * CH + (chunk ^ k_swizzle(row & 15))] = u32x4{k0[0], k0[1], k1[0], k1[1]};
        kv[buf][1][row * CH + (chunk ^ v_swizzle(row))] = u32x4{v0[0], v0[1], v1[0], v1[1]};
      }
      if (C::kPasses && __builtin_expect(top_of(raw_ks, vs) >= kMostBits, 0))
#pragma unroll 1
        for (int c = 0; c < 2 * CH / 8; ++c) {  // as they lie in LDS, eight threads to a row
          const bool keys = c < CH / 8;
          const int chunk = part * (CH / 8) + c % (CH / 8);
          u32x4& x = kv[buf][keys ? 0 : 1]
                       [row * CH + (chunk ^ (keys ? k_swizzle(row & 15) : v_swizzle(row)))];
          x = at_most(x);
        }
      if ((wave & 1) == 0 && lane == 0) marks[buf][tile] = (wild ? 1 : 0) | (raw_out ? 4 : 0);
    };
    __syncthreads();  // the last segment's reads are done
    if (seg.t0 < t1) load(seg.t0);
    r.load_q(y.a, seg, r0, n16, g4);
    r.clear();
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, 1> second;
    if (seg.t0 < t1) store(first);
    if (seg.t0 + 1 < t1) load(seg.t0 + 1);
    auto step = [&](int t, auto buffer, auto other) {
      constexpr int buf = buffer;
      const int k0 = t * kStep;
      __syncthreads();  // this step's keys are there, those of the step before have been read
      if (t + 1 < t1) store(other);
      if (t + 2 < t1) load(t + 2);
      if (k0 >= r.hi || r0 >= rows) return;
      const u32x4* const ks = kv[buf][0];
      const u32x4* const vs = kv[buf][1];
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
      const int mark = uniform(marks[buf][0] | marks[buf][1] << 1);
      if (k0 + kStep > r.lo || mark >> 2) {
        const int n[2] = {tile_of(y, view, k0).n, tile_of(y, view, k0 + 16).n};
        r.mask(sc, vr, n, k0, g4);
      }
      u32x4 ph[NT], pl[NT];
      r.weights(sc, y.a.c, ph, pl);
      r.product(vr, ph, pl);
      // here, after the products: ahead of them their sums took other registers, and a move each
      if (mark & 3) spoil(r, mark, k0);
    };
    for (int t = seg.t0; t < t1; t += 2) {
      step(t, first, second);
      if (t + 1 < t1) step(t + 1, second, first);
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
  return launch_join_many<D, NT, ManyDeal>(x.a, st);
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
  return launch_join_few<D, Few8Deal>(x.a, st);
}

}  // namespace
}  // namespace umic

extern "C" int64_t umic_cache8_attention_workspace_bytes(int64_t S, int64_t Hq, int64_t Hk,
                                                         int64_t D) {
  return umic::workspace_bytes(S, Hq, Hk, D, umic::few8_of(D));
}

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
  if (const int e = attn_args(call, 16, few8_of(D), x.a, s)) return e == 1 ? UMIC_OK : e;
  // Single tokens of up to a sixteenth of the CUs' segments, and less than five units for
  // two workgroups a CU: one, half the parts (8 segments of 12288 keys 13.1 us for 15.6, 16
  // of 3500 21 for 28; 32 of 4000 14.0 for 13.5, 8 of 131072 60 for 53).
  const int cus = s.nwg / few8_of(D);
  if (s.nt == 0 && B * c.heads * 16 <= cus) x.a.some = cus;
  x.ks = c.k_scale, x.vs = c.v_scale, x.s_sb = c.s_sb, x.s_sh = c.s_sh;
  hipStream_t st = as_stream(stream);
  const bool f = c.format == UMIC_CODES_INT8;
  if (D == 64)
    return f ? launch8<64, UMIC_CODES_INT8>(s, x, st) : launch8<64, UMIC_CODES_E4M3>(s, x, st);
  if (D == 128)
    return f ? launch8<128, UMIC_CODES_INT8>(s, x, st) : launch8<128, UMIC_CODES_E4M3>(s, x, st);
  return f ? launch8<256, UMIC_CODES_INT8>(s, x, st) : launch8<256, UMIC_CODES_E4M3>(s, x, st);
}
