// A paged key / value cache in 8 bits: new tokens' rows rotated and written as codes, and
// rows read back as bf16.
//
// A block is 16 consecutive rows of a page, of one key head.  With a = max |x| over the
// values that come into it, its scale is s = 2^e, e = floor(log2 a) - 6 (int8) or - 7
// (e4m3), and at least what it was where the block holds tokens already; its codes are
// x / s to the nearest, ties to even.  Where the scale grows, the codes of the rows before
// are rounded to it: it at least doubles, so that all roundings of such a row are within
// half a step of the last scale and a half of that, and so on: one step.  The scale is
// that of bf16 values' exponents, whole numbers throughout.
//
// A block is its first token's workgroup's to write, with all tokens that the call brings to
// it.  A wave finds them by its lanes where they stand within kSpan neighbours, and 16 there
// are all.  Of a block with fewer the workgroup looks through all slots of the call, 8 bytes
// a token: tokens before the first one make it another's, and with others behind it the block
// is done by itself, after the rest.  A prompt has two such blocks, at its ends, and single
// tokens have no others.  (64 of them 6.3 us, 6.1 without the look; 16384 tokens of one
// request 63 and 63, without a rotation, which hides some of it, 29 and 25.)  Behind those
// workgroups stand others that rotate q.
//
// What bounds it: HBM at prompt sizes, 16381 tokens of 32 + 8 heads of 128 62 us, 5.9 TB/s
// (a large copy 6.1); 3100 with the norm 19.3, of which 12 are their bytes', the rest the
// chain of a block (its slots, rows, maximum, codes); 8 tokens 6, that chain alone.
#include "axial.hpp"
#include "codes.hpp"

namespace umic {
namespace {

constexpr int kWaves = kThreads / kWave;
constexpr int kSpan = 24;    // tokens among which a wave finds a block's by its lanes
constexpr int kChunk = 16;   // tokens of a workgroup, at most
static_assert(kChunk + 2 * (kSpan - 1) <= kWave, "a wave sees a chunk and its neighbours");
constexpr int kEarlier = 1 << 16;  // counts a block's tokens before the first one near

struct StoreArgs {
  AxialArgs x;  // of q's rows: Hq heads, no keys; and what k's rotation needs
  const uint16_t* k;
  const uint16_t* v;
  uint8_t* k8;
  uint8_t* v8;
  float* ks;
  float* vs;
  int64_t Hk, k_st, k_sh, v_st, v_sh;
  int64_t c_sb, c_sh, c_ss, s_sb, s_sh;
  int64_t slots_n;
  int shift;         // of a page
  int chunk;         // tokens of a workgroup: it does the blocks whose first is among them
  int split;         // workgroups of a chunk, which share its blocks' heads
  unsigned blocks;   // workgroups that do so; those behind them rotate q
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// x of another lane; all lanes are there.
__device__ __forceinline__ int of_lane(int x, int lane) {
  return __builtin_amdgcn_ds_bpermute(lane * 4, x);
}

__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const u16x2 m = __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b));
  return __builtin_bit_cast(uint32_t, m);
}

// f over 16 neighbouring lanes, by moves of the vector unit: with shuffles, whose lane numbers
// take a register each, the blocks done one by one did not fit.
template <typename F>
__device__ __forceinline__ int over16(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, false));  // row_half_mirror
  return f(x, __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, false));  // row_mirror
}

// The kernel's arguments, loaded again: what the rare paths need of them is not held over the
// others.
__device__ __forceinline__ StoreArgs store_args_again() {
  typedef const __attribute__((address_space(4))) StoreArgs* Args;
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const StoreArgs*)p;
}

// A wave's task is a block's new tokens of one head, keys or values.  The sines and cosines
// are the workgroup's, once for all heads.
template <int D, int FORMAT, bool TURN, bool NORM>
__global__ __launch_bounds__(kThreads, D <= 128 ? 4 : 2) void store_kernel(StoreArgs a) {
  typedef Codes<FORMAT> C;
  constexpr int kLanes = D / 16;            // of a row, 8 elements of each half a lane
  constexpr int kRows = kWave / kLanes;     // rows of a pass
  constexpr int kPasses = kBlockTokens / kRows;
  constexpr int kOld = D / 64;              // 16-byte chunks of a block's codes a lane holds
  constexpr int kTurns = 2 * kThreads / D;  // tokens whose sines the workgroup does at a time
  extern __shared__ float cs[];             // (cos, sin): [token][pair]
  __shared__ int far_n[kChunk];             // tokens of a block that are not near its first one
  __shared__ int far[kChunk][kBlockTokens];
  __shared__ int found[kWaves];             // a wave has seen such tokens
  if (blockIdx.x >= a.blocks) {
    if constexpr (TURN) axial_rows<8, NORM, (D >= 128), true>(a.x, blockIdx.x - a.blocks, cs);
    return;
  }
  const int lane = threadIdx.x & (kWave - 1);
  const int waves = kWaves * a.split, parts = 2 * (int)a.Hk;
  // Chunks in another order than workgroups: the first, then from the last one on, as a prompt's
  // ends look through all slots, and what begins last ends the launch; and each 64 of them turned
  // by another number of places, as ends of requests of one length are a power of two chunks
  // apart, and in order all on a few CUs (16384 tokens of 64 requests of 256: 63 us for 77).
  const unsigned chunks = a.blocks / a.split, nth_one = blockIdx.x / a.split;
  unsigned chunk = nth_one ? chunks - nth_one : 0;
  if ((chunk | 63) < chunks) chunk = (chunk & ~63u) | ((chunk + (chunk >> 6) * 37) & 63);
  const int64_t t0 = (int64_t)chunk * a.chunk;
  const int mine = uniform(blockIdx.x % a.split * kWaves + threadIdx.x / kWave);

  // lane i: token t0 - (kSpan - 1) + i, its block and row; a slot outside the pool has none
  const int64_t base = t0 - (kSpan - 1);
  auto slot_of = [&](const StoreArgs& a, int lane) {
    const int64_t tok = base + lane;
    const bool in = lane < a.chunk + 2 * (kSpan - 1) && tok >= 0 && tok < a.x.T;
    return in ? a.x.slots[tok] : -1;
  };
  const int64_t slot = slot_of(a, lane);
  // The look through all slots: few are asked for here, beside the lanes' own.  (After them
  // 64 single tokens took 7.0 us.)
  const bool wide = a.x.T > kSpan;  // no two tokens of fewer are further apart
  constexpr int kPairs = 4;         // of slots, a thread's at a time
  typedef int64_t pair_t __attribute__((ext_vector_type(2), aligned(8)));
  constexpr int kLook = kPairs * 2 * kThreads;
  auto token_of = [](int64_t i, int u) { return i + u * 2 * kThreads + threadIdx.x * 2; };
  auto load_slots = [&](const StoreArgs& a, int64_t i, pair_t (&p)[kPairs]) {
#pragma unroll
    for (int u = 0; u < kPairs; ++u)  // past the end the last pair again
      p[u] = *reinterpret_cast<const pair_t*>(a.x.slots + min(token_of(i, u), a.x.T - 2));
  };
  const bool few = a.x.T <= kLook;
  pair_t ahead[kPairs];
  if (wide && few) load_slots(a, 0, ahead);
  int axis = -1;
  uint64_t turn = 0;
  if constexpr (TURN) {
    axis = a.x.axis[threadIdx.x % (D / 2)];
    turn = a.x.turn[threadIdx.x % (D / 2)];
  }
  auto block_of = [](const StoreArgs& a, int64_t slot) {
    return slot >= 0 && slot < a.slots_n ? (int)(slot / kBlockTokens) : -1;
  };
  int block = block_of(a, slot), row = (int)(slot & (kBlockTokens - 1)), where = lane;
  // lane i: where the i-th of some of the lanes stands
  auto nth = [&](uint64_t some) {
    const int below =
        __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
    const int to = some >> lane & 1 ? below : __builtin_popcountll(some) + lane - below;
    return __builtin_amdgcn_ds_permute(to * 4, lane);
  };
  // the tokens of lane at's block that stand near it
  auto near_of = [&](int at) {
    const int blk = __builtin_amdgcn_readlane(block, at);
    return __ballot(block == blk) >> at << (64 - kSpan) >> (64 - kSpan) << at;
  };

  // Of the chunk's tokens: those that are their block's first, and those of them whose block
  // can have more than the ones near; and all tokens near a first.
  uint32_t now = 0, open = 0;
  uint64_t all = 0;
  bool more = false;  // some has
  for (int c = 0; c < a.chunk; ++c) {
    const int at = kSpan - 1 + c;
    const int blk = __builtin_amdgcn_readlane(block, at);
    const uint64_t mates = __ballot(block == blk);
    // a block is its first token's to write
    if (blk < 0 || mates << (64 - at)) continue;
    const uint64_t run = near_of(at);
    now |= 1u << c;
    all |= run;
    if (__builtin_popcountll(run) < kBlockTokens) open |= 1u << c;
    if (mates != run) more = true;
  }
  if (!now) return;
  if (!wide) open = 0;
  if (open) {
    if (!few) load_slots(a, 0, ahead);
    for (int64_t i = 0; i < a.x.T; i += kLook) {
      uint32_t blk[2 * kPairs];  // without the bits above: one may seem to be a block's that is
                                 // not, and gather() looks again
#pragma unroll
      for (int u = 0; u < kPairs; ++u)
        for (int v = 0; v < 2; ++v) blk[2 * u + v] = (uint32_t)((uint64_t)ahead[u][v] / kBlockTokens);
      if (i + kLook < a.x.T) load_slots(a, i + kLook, ahead);
      if (i < base + kWave && i + kLook > base)  // the neighbours have been looked at
#pragma unroll
        for (int u = 0; u < 2 * kPairs; ++u) {
          const int64_t t = min(token_of(i, u >> 1), a.x.T - 2) + (u & 1);
          if ((uint64_t)(t - base) < (uint64_t)(a.chunk + 2 * (kSpan - 1))) blk[u] = ~0u;
        }
#pragma unroll 1
      for (uint32_t m = open; m; m &= m - 1) {
        const uint32_t its = __builtin_amdgcn_readlane(block, kSpan - 1 + __builtin_ctz(m));
#pragma unroll
        for (int u = 0; u < 2 * kPairs; ++u) more |= blk[u] == its;
      }
    }
    const bool any = __any(more);
    if (lane == 0) found[threadIdx.x / kWave] = any;
  }
  uint32_t apart = 0;  // firsts whose blocks have tokens that are not near them
  // Tokens that are not near their block's first one: the block is another workgroup's, or apart.
  auto gather = [&] {
    const StoreArgs z = store_args_again();
    if (threadIdx.x < kChunk) far_n[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll 1
    for (int64_t i = 0; i < z.x.T; i += kLook) {
      load_slots(z, i, ahead);
#pragma unroll 1
      for (uint32_t m = open; m; m &= m - 1) {
        const int c = __builtin_ctz(m), its = __builtin_amdgcn_readlane(block, kSpan - 1 + c);
#pragma unroll
        for (int u = 0; u < 2 * kPairs; ++u) {
          const int64_t t = token_of(i, u >> 1) + (u & 1), off = t - base - (kSpan - 1 + c);
          // of the last pair for an odd one out, its second slot
          const int64_t slot = ahead[u >> 1][t == z.x.T - 1 && !(u & 1) ? 1 : u & 1];
          if (t >= z.x.T || block_of(z, slot) != its || (off >= 0 && off < kSpan)) continue;
          const int n = atomicAdd(&far_n[c], off < 0 ? kEarlier : 1) & (kEarlier - 1);
          if (off > 0 && n < kBlockTokens) far[c][n] = (int)(t - base);
        }
      }
    }
    __syncthreads();
    for (uint32_t m = open; m; m &= m - 1) {
      const int n = uniform(far_n[__builtin_ctz(m)]);
      if (!n) continue;
      now &= ~(m & -m);
      if (n < kEarlier) apart |= m & -m;
    }
  };
  const int c8 = (lane % kLanes) * 8;
  // the blocks whose tokens are near, then the others one by one
  for (bool first = true;; first = false) {
    if (__builtin_expect(!now, 0)) {
      if (!apart) break;
      const StoreArgs z = store_args_again();
      const int c = __builtin_ctz(apart), at = kSpan - 1 + c;
      now = apart & -apart;
      apart &= apart - 1;
      // lanes at .. get the block's tokens
      int again = lane;
      asm volatile("" : "+v"(again));  // what follows from it is not held over the tasks
      block = block_of(z, slot_of(z, again));
      const uint64_t run = near_of(at);
      const int near = __builtin_popcountll(run);
      const int n = min(kBlockTokens, near + uniform(far_n[c]));
      const int i = lane - at;
      where = of_lane(nth(run), i & (kWave - 1));
      if (i >= near && i < n) where = far[c][i - near];
      block = -1;
      if (i >= 0 && i < n) {
        const int64_t slot = z.x.slots[base + where];
        block = block_of(z, slot);
        row = (int)(slot & (kBlockTokens - 1));
      }
      all = __ballot(block >= 0);
      if (TURN) __syncthreads();  // the sines have been read
    }
    if constexpr (TURN) {
      const int turned = of_lane(where, nth(all)), count = __builtin_popcountll(all);
      const bool moves = axis >= 0 && axis < a.x.A;  // an axis that is not there does not turn
      constexpr int kAhead = 4;                      // positions on their way
      int thread = threadIdx.x;
      asm volatile("" : "+v"(thread));  // as above
      for (int i = 0; i < count; i += kAhead * kTurns) {
        int64_t pos[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int t = i + u * kTurns + thread / (D / 2);
          const int64_t token = base + of_lane(turned, min(t, count - 1));
          pos[u] = moves ? a.x.positions[axis * a.x.p_sa + token * a.x.p_st] : 0;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int t = i + u * kTurns + thread / (D / 2);
          if (i + u * kTurns >= count) break;
          float s, c;
          turn_of<true>(pos[u], turn, s, c);
          if (t < count)
            *reinterpret_cast<f32x2_t*>(cs + t * D + turn_at(thread % (D / 2), kLanes)) =
                f32x2_t{c * a.x.scale, s * a.x.scale};
        }
      }
    }
    if (TURN || (first && open)) __syncthreads();
    if (first && open && __builtin_expect(uniform(found[0] | found[1] | found[2] | found[3]), 0))
      gather();

    int part = mine;
    for (; now; now &= now - 1, part -= parts) {
      // the chunk's tasks, its blocks' parts in turn, are dealt over the waves
      if (part >= parts) continue;
      const int at = kSpan - 1 + __builtin_ctz(now);
      const int blk = __builtin_amdgcn_readlane(block, at);
      const uint64_t run = near_of(at);
      const int n = min(kBlockTokens, __builtin_popcountll(run));
      const int place = nth(run);
      const int its_row = of_lane(row, place), its_where = of_lane(where, place);
      const int its_turn = __builtin_popcountll(all & (((uint64_t)1 << place) - 1));
      int row0 = lane < n ? its_row : kBlockTokens;  // the lowest
      row0 = uniform(over16(row0, [](int x, int y) { return min(x, y); }));
      const int64_t in_pool = (int64_t)blk * kBlockTokens;
      const int64_t page = in_pool >> a.shift;
      const int64_t r0 = in_pool & (((int64_t)1 << a.shift) - 1);
      int at_row[kPasses];  // its row, and times 16 where its sines are; negative: no token
      int of[kPasses];      // where it stands
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int i = lane / kLanes + p * kRows;
        of[p] = of_lane(its_where, i);
        at_row[p] = of_lane(its_turn * kBlockTokens + its_row, i);
        if (i >= n) at_row[p] = (int)0x80000000;
      }
      u32x4 lo[kPasses], hi[kPasses];
      auto fetch = [&](int part) {
        const bool keys = part < a.Hk;
        const int h = keys ? part : part - (int)a.Hk;
        const uint16_t* const src = (keys ? a.k : a.v) + h * (keys ? a.k_sh : a.v_sh) + c8;
        const int64_t st = keys ? a.k_st : a.v_st;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          lo[p] = hi[p] = u32x4{0, 0, 0, 0};
          if (at_row[p] >= 0) {
            const uint16_t* x = src + (base + of[p]) * st;
            lo[p] = ld_stream(reinterpret_cast<const u32x4*>(x));
            hi[p] = ld_stream(reinterpret_cast<const u32x4*>(x + D / 2));
          }
        }
      };
      fetch(part);
#pragma unroll 1
      for (; part < parts; part += waves) {
        const bool keys = part < a.Hk;
        const int h = keys ? part : part - (int)a.Hk;
        const StoreArgs y = store_args_again();
        uint8_t* const to = (keys ? y.k8 : y.v8) + page * y.c_sb + h * y.c_sh + r0 * y.c_ss;
        float* const scale = (keys ? y.ks : y.vs) + page * y.s_sb + h * y.s_sh + r0 / kBlockTokens;
        u32x4 old[kOld];
        float was = 0.0f;
        if (row0 > 0) {
          was = *scale;
#pragma unroll
          for (int j = 0; j < kOld; ++j) {
            const int i = j * kWave + lane, r = i / (D / 16);
            old[j] = u32x4{0, 0, 0, 0};
            if (r < row0) old[j] = *reinterpret_cast<const u32x4*>(to + r * y.c_ss + i % (D / 16) * 16);
          }
        }
        if constexpr (TURN)
          if (keys)
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
              if (p * kRows >= n) break;
              float x[8], y[8], ox[8], oy[8];
              unpack8(lo[p], x);
              unpack8(hi[p], y);
              if constexpr (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += x[j] * x[j] + y[j] * y[j];
                const float r = rsqrt_cr(group_sum<kLanes>(ss) / (float)D + a.x.eps);
                auto by = [&](float (&z)[8], const uint16_t* w) {
                  float f[8];
                  unpack8(*reinterpret_cast<const u32x4*>(w), f);
#pragma unroll
                  for (int j = 0; j < 8; ++j) z[j] = z[j] * r * f[j];
                };
                by(x, a.x.kw + c8);
                __builtin_amdgcn_sched_barrier(0);  // both halves' weights at once do not fit
                by(y, a.x.kw + c8 + D / 2);
              }
              const float* t = cs + (at_row[p] & 0xffff) / kBlockTokens * D + c8 / 2;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float* cosine = t + (j >> 1) * (4 * kLanes) + (j & 1) * 2;
                ox[j] = x[j] * cosine[0] - y[j] * cosine[1];
                oy[j] = y[j] * cosine[0] + x[j] * cosine[1];
              }
              const bool is = at_row[p] >= 0;
              lo[p] = is ? pack8(ox) : u32x4{0, 0, 0, 0};
              hi[p] = is ? pack8(oy) : u32x4{0, 0, 0, 0};
            }
        // the largest magnitude's exponent: that of bf16 numbers as whole ones
        uint32_t top = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            top = max_halves(top, max_halves(lo[p][w] & 0x7fff7fffu, hi[p][w] & 0x7fff7fffu));
        top = over16((int)top, [](int x, int y) { return (int)max_halves(x, y); });
        const int one = (int)max(top & 0xffffu, top >> 16);
        const int most = max(max(__builtin_amdgcn_readlane(one, 0), __builtin_amdgcn_readlane(one, 16)),
                             max(__builtin_amdgcn_readlane(one, 32), __builtin_amdgcn_readlane(one, 48)));
        const uint32_t was_bits = __builtin_amdgcn_readfirstlane(__float_as_uint(was));
        // 255: infinite or NaN; the block then reads as NaN
        const bool wild = (most >> 7) == 255 || (row0 > 0 && (was_bits << 1) >= 0xff000000u);
        const int was_exp = (int)(was_bits >> 23 & 255) - 127;
        int e = max((most >> 7) - 127 - C::kTop, kLeastExp);
        if (row0 > 0) e = max(e, was_exp);
        const float s = __uint_as_float((uint32_t)(e + 127) << 23);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        if (lane == 0) *scale = wild ? __builtin_nanf("") : s;
        uint32_t w[kPasses][4];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          float x[8], y[8];
          unpack8(lo[p], x);
          unpack8(hi[p], y);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= inv, y[j] *= inv;
          w[p][0] = C::round4(x), w[p][1] = C::round4(x + 4);
          w[p][2] = C::round4(y), w[p][3] = C::round4(y + 4);
        }
        if (part + waves < parts) fetch(part + waves);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          if (at_row[p] < 0) continue;
          uint8_t* r = to + (at_row[p] & (kBlockTokens - 1)) * y.c_ss + c8;
          *reinterpret_cast<u32x2*>(r) = wild ? u32x2{0, 0} : u32x2{w[p][0], w[p][1]};
          *reinterpret_cast<u32x2*>(r + D / 2) = wild ? u32x2{0, 0} : u32x2{w[p][2], w[p][3]};
        }
        if (row0 > 0 && !wild && e > was_exp) {  // the rows before, at the new scale
          const float ratio = was * inv;
#pragma unroll
          for (int j = 0; j < kOld; ++j) {
            const int i = j * kWave + lane, r = i / (D / 16);
            if (r >= row0) continue;
            u32x4 o;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float x[4];
              C::values4(old[j][q], x);
#pragma unroll
              for (int y = 0; y < 4; ++y) x[y] *= ratio;
              o[q] = C::round4(x);
            }
            *reinterpret_cast<u32x4*>(to + r * y.c_ss + i % (D / 16) * 16) = o;
          }
        }
      }
    }
  }
}

struct ReadArgs {
  const uint8_t* k8;
  const uint8_t* v8;
  const float* ks;
  const float* vs;
  uint16_t* ko;
  uint16_t* vo;
  const int32_t* table;
  const int32_t* kv_len;  // or NULL: len
  const int32_t* start;   // or NULL: 0
  int64_t c_sb, c_sh, c_ss, s_sb, s_sh, table_ld;
  int64_t rows, blocks;
  int len, cap, shift, pages, Hk;
};

// A scalar load whatever the compiler can prove about the kernel's stores.
__device__ __forceinline__ int scalar_i32(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

// A thread's 8 codes at a time to 16 bytes, in ITEMS rows whose loads are on their way
// together.  HBM-bound: 4 x 30011 rows of 8 heads of 128 119.9 us, 6.2 TB/s (one row a
// thread 156, four 127, 16 codes to two stores 129); of padded rows, mostly zeros, 166 MB
// in 31 us (one 33, four 34).
template <int D, int FORMAT, int ITEMS>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  typedef Codes<FORMAT> C;
  constexpr int kChunks = D / 8, kRows = kThreads / kChunks;
  const int64_t head = blockIdx.x / (unsigned)a.blocks;  // (request, k or v, key head)
  const unsigned block = blockIdx.x % (unsigned)a.blocks;
  const int h = (int)((unsigned)head % (unsigned)a.Hk);
  const unsigned rest = (unsigned)head / (unsigned)a.Hk;
  const int b = (int)(rest >> 1);
  const bool keys = !(rest & 1);
  const int c = threadIdx.x % kChunks * 8;
  const int64_t row0 = (int64_t)block * (ITEMS * kRows) + threadIdx.x / kChunks;
  const int n = a.kv_len ? min(max(scalar_i32(a.kv_len + b), 0), a.cap) : a.len;
  const int64_t at0 = row0 + (a.start ? max(scalar_i32(a.start + b), 0) : 0);
  const uint8_t* const codes = (keys ? a.k8 : a.v8) + h * a.c_sh + c;
  const float* const scales = (keys ? a.ks : a.vs) + h * a.s_sh;
  const int32_t* const table = a.table + b * a.table_ld;
  int page[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = at0 + i * kRows;
    page[i] = at < n ? table[at >> a.shift] : -1;
  }
  u32x2 w[ITEMS];
  float s[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t in = (at0 + i * kRows) & (((int64_t)1 << a.shift) - 1);
    w[i] = u32x2{0, 0};
    s[i] = 0.0f;
    if ((unsigned)page[i] < (unsigned)a.pages) {  // others are not there
      w[i] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x2*>(codes + page[i] * a.c_sb + in * a.c_ss));
      s[i] = scales[page[i] * a.s_sb + in / kBlockTokens];
    }
  }
  uint16_t* const to =
      (keys ? a.ko : a.vo) + (((int64_t)b * a.Hk + h) * a.rows + row0) * D + c;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (row0 + i * kRows >= a.rows) break;
    float x[4], y[4];
    C::values4(w[i][0], x);
    C::values4(w[i][1], y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= s[i], y[j] *= s[i];
    if (C::kPasses && s[i] >= kMostScale)
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // not fminf: NaN stays
        x[j] = x[j] > kMost ? kMost : x[j] < -kMost ? -kMost : x[j];
        y[j] = y[j] > kMost ? kMost : y[j] < -kMost ? -kMost : y[j];
      }
    st_stream(reinterpret_cast<u32x4*>(to + (int64_t)i * kRows * D),
              u32x4{pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(y[0], y[1]), pack2(y[2], y[3])});
  }
}

template <int D, int FORMAT>
int launch_store(StoreArgs& a, bool turn, hipStream_t st) {
  unsigned grid = 0;
  size_t lds = 0;
  if (turn && a.x.Hq) {
    AxialShape s;
    if (const int e = axial_shape(a.x, s)) return e;
    if (s.vec != 8) return UMIC_ERR_UNSUPPORTED;
    grid = s.blocks;
    lds = s.lds;
  }
  const int64_t cus = device_cus();
  if (cus <= 0) return (int)hipErrorNoDevice;
  // Two chunks to a CU's workgroup in four, up to kChunk tokens each; then a workgroup for
  // each four tasks of a block while there are not two to a CU.  (Chunks of a token up to
  // 2048 of them: 42 us for 16.5, most workgroups having no block's first token; four times
  // the chunks 20.9.  Four workgroups to a CU: 3100 tokens 23.7 us for 19.0, and one 19.4,
  // where 4096 tokens of 64 requests take 39 for 29.)
  a.chunk = (int)std::min<int64_t>((2 * a.x.T + cus - 1) / cus, kChunk);
  const int64_t chunks = (a.x.T + a.chunk - 1) / a.chunk;
  a.split = (int)std::max<int64_t>(
      1, std::min<int64_t>((2 * a.Hk + kWaves - 1) / kWaves, 2 * cus / chunks));
  if (turn)
    lds = std::max(lds, (size_t)std::min(a.chunk + kSpan - 1, a.chunk * kSpan) * D * sizeof(float));
  const int64_t blocks = chunks * a.split;
  if (blocks + grid > 0x7fffffff) return UMIC_ERR_UNSUPPORTED;
  a.blocks = (unsigned)blocks;
  auto* kern = !turn    ? store_kernel<D, FORMAT, false, false>
               : a.x.kw ? store_kernel<D, FORMAT, true, true>
                        : store_kernel<D, FORMAT, true, false>;
  hipLaunchKernelGGL(kern, dim3(a.blocks + grid), dim3(kThreads), lds, st, a);
  return launch_status();
}

template <int D, int FORMAT>
int launch_read(ReadArgs& a, int64_t heads, hipStream_t st) {
  constexpr int kItems = 2, kRows = kThreads / (D / 8);
  const int64_t cus = device_cus();
  if (cus <= 0) return (int)hipErrorNoDevice;
  // Two rows a thread where that leaves eight workgroups to a CU; fewer would not fill it.
  const bool many = (a.rows + kItems * kRows - 1) / (kItems * kRows) * heads >= 8 * cus;
  const int64_t per = kRows * (many ? kItems : 1);
  a.blocks = (a.rows + per - 1) / per;
  if (a.blocks > 0x7fffffff / heads) return UMIC_ERR_UNSUPPORTED;
  auto* kern = many ? read_kernel<D, FORMAT, kItems> : read_kernel<D, FORMAT, 1>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.blocks * heads)), dim3(kThreads), 0, st, a);
  return launch_status();
}

}  // namespace

int check_cache8(const umic_cache8_t* c, int64_t& cap, int64_t table_w) {
  if (!c || c->pages < 0 || c->page_size <= 0 || c->heads <= 0 || c->head_dim <= 0 || table_w < 0)
    return UMIC_ERR_INVALID_ARG;
  if (c->pages && (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale))
    return UMIC_ERR_INVALID_ARG;
  const int64_t D = c->head_dim, ps = c->page_size;
  if ((D != 64 && D != 128 && D != 256) || ps < 16 || (ps & (ps - 1)) || ps > ((int64_t)1 << 30) ||
      c->pages > ((int64_t)1 << 30) || c->pages * ps > ((int64_t)1 << 34) ||
      table_w > ((int64_t)1 << 30) / ps || c->heads > (1 << 16) ||
      (c->format != UMIC_CODES_E4M3 && c->format != UMIC_CODES_INT8))
    return UMIC_ERR_UNSUPPORTED;
  if (((c->c_sb | c->c_sh | c->c_ss) & 15) || !aligned16(c->k_codes) || !aligned16(c->v_codes))
    return UMIC_ERR_UNSUPPORTED;
  cap = c->pages ? table_w * ps : 0;
  return UMIC_OK;
}

}  // namespace umic

extern "C" int umic_cache8_append_bf16(
    const umic_cache8_t* cache, const void* q, const void* k, const void* v, void* q_out,
    const int64_t* positions, const uint64_t* turn, const int32_t* axis, const int64_t* slots,
    float scale, const void* q_w, const void* k_w, float eps, int64_t T, int64_t Hq, int64_t axes,
    int64_t p_sa, int64_t p_st, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
    int64_t v_st, int64_t v_sh, void* stream) {
  using namespace umic;
  int64_t cap;
  if (const int e = check_cache8(cache, cap, 0)) return e;
  if (T < 0 || Hq < 0) return UMIC_ERR_INVALID_ARG;
  if (T == 0) return UMIC_OK;
  if (!k || !v || !slots) return UMIC_ERR_INVALID_ARG;
  if (turn) {
    if (axes <= 0 || !positions || !axis || (Hq && (!q || !q_out)) || (!q_w != !k_w))
      return UMIC_ERR_INVALID_ARG;
  } else if (Hq || q_w || k_w) {
    return UMIC_ERR_INVALID_ARG;
  }
  if (T > 0x7fffffff || Hq > (1 << 16) || ((q_st | q_sh | k_st | k_sh | v_st | v_sh) & 7) ||
      !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(q_w) || !aligned16(k_w))
    return UMIC_ERR_UNSUPPORTED;
  const umic_cache8_t& c = *cache;
  const int64_t D = c.head_dim;
  StoreArgs a = {};
  a.x.q = (const uint16_t*)q, a.x.qo = (uint16_t*)q_out;
  a.x.positions = positions, a.x.turn = turn, a.x.axis = axis, a.x.slots = slots;
  a.x.qw = (const uint16_t*)q_w, a.x.kw = (const uint16_t*)k_w;
  a.x.T = T, a.x.Hq = Hq, a.x.D = D, a.x.A = axes, a.x.p_sa = p_sa, a.x.p_st = p_st;
  a.x.q_st = q_st, a.x.q_sh = q_sh, a.x.qo_st = Hq * D, a.x.qo_sh = D;
  a.x.eps = eps, a.x.scale = scale;
  a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.k8 = (uint8_t*)c.k_codes, a.v8 = (uint8_t*)c.v_codes, a.ks = c.k_scale, a.vs = c.v_scale;
  a.Hk = c.heads, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  a.c_sb = c.c_sb, a.c_sh = c.c_sh, a.c_ss = c.c_ss, a.s_sb = c.s_sb, a.s_sh = c.s_sh;
  a.slots_n = c.pages * c.page_size;
  a.shift = __builtin_ctzll((unsigned long long)c.page_size);
  hipStream_t st = as_stream(stream);
  const bool t = turn != nullptr, f = c.format == UMIC_CODES_INT8;
  if (D == 64)
    return f ? launch_store<64, UMIC_CODES_INT8>(a, t, st) : launch_store<64, UMIC_CODES_E4M3>(a, t, st);
  if (D == 128)
    return f ? launch_store<128, UMIC_CODES_INT8>(a, t, st)
             : launch_store<128, UMIC_CODES_E4M3>(a, t, st);
  return f ? launch_store<256, UMIC_CODES_INT8>(a, t, st) : launch_store<256, UMIC_CODES_E4M3>(a, t, st);
}

extern "C" int umic_cache8_read_bf16(const umic_cache8_t* cache, void* k_out, void* v_out,
                                     const int32_t* table, const int32_t* kv_lens,
                                     const int32_t* starts, int64_t B, int64_t rows,
                                     int64_t table_ld, int64_t table_w, int64_t kv_len,
                                     void* stream) {
  using namespace umic;
  int64_t cap;
  if (const int e = check_cache8(cache, cap, table_w)) return e;
  if (B < 0 || rows < 0 || table_ld < table_w) return UMIC_ERR_INVALID_ARG;
  if (B == 0 || rows == 0) return UMIC_OK;
  if (!k_out || !v_out || !table) return UMIC_ERR_INVALID_ARG;
  if (!kv_lens && (kv_len < 0 || kv_len > cap)) return UMIC_ERR_INVALID_ARG;
  if (B > (1 << 20) || 2 * B * cache->heads > 0x7fffffff || rows > ((int64_t)1 << 31) ||
      !aligned16(k_out) || !aligned16(v_out))
    return UMIC_ERR_UNSUPPORTED;
  const umic_cache8_t& c = *cache;
  const int64_t D = c.head_dim;
  ReadArgs a = {};
  a.k8 = (const uint8_t*)c.k_codes, a.v8 = (const uint8_t*)c.v_codes;
  a.ks = c.k_scale, a.vs = c.v_scale;
  a.ko = (uint16_t*)k_out, a.vo = (uint16_t*)v_out;
  a.table = table, a.kv_len = kv_lens, a.start = starts;
  a.c_sb = c.c_sb, a.c_sh = c.c_sh, a.c_ss = c.c_ss, a.s_sb = c.s_sb, a.s_sh = c.s_sh;
  a.table_ld = table_ld, a.rows = rows, a.len = (int)kv_len, a.cap = (int)cap;
  a.shift = __builtin_ctzll((unsigned long long)c.page_size);
  a.pages = (int)c.pages, a.Hk = (int)c.heads;
  const int64_t heads = 2 * B * c.heads;
  hipStream_t st = as_stream(stream);
  const bool f = c.format == UMIC_CODES_INT8;
  if (D == 64)
    return f ? launch_read<64, UMIC_CODES_INT8>(a, heads, st)
             : launch_read<64, UMIC_CODES_E4M3>(a, heads, st);
  if (D == 128)
    return f ? launch_read<128, UMIC_CODES_INT8>(a, heads, st)
             : launch_read<128, UMIC_CODES_E4M3>(a, heads, st);
  return f ? launch_read<256, UMIC_CODES_INT8>(a, heads, st)
           : launch_read<256, UMIC_CODES_E4M3>(a, heads, st);
}
