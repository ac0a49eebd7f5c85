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
#include "attention.hpp"

namespace umic {
namespace {

// Up to 16 rows: a wave takes 32 of a tile's 128 keys.  The loads of a step are in
// flight while the one before is computed, and the next segment's first while the
// waves of this one are joined.
constexpr int few_of(int64_t D) { return D <= 128 ? 2 : 1; }

template <int D>
__global__ __launch_bounds__(kThreads, few_of(D)) void attend_few_kernel(AttnArgs a) {
  typedef Rows<D, 1, false> R;
  constexpr int KK = R::KK, DV = R::DV, VW = R::VW;
  constexpr int kTile = kStep * kWaves;
  __shared__ FewShared<D> lds;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;

  Scan scan = {};
  const int even = a.kv_len ? 0 : FewDeal::units(a.len);  // units of each, if all have as many
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

      join_waves<D, true>(args_again(), r, seg, lds, wg, split);
      seg = nxt;
    }
    const AttnArgs args = args_again();
    join_parts<D>(args, deal, lds, split);
  }
  const AttnArgs z = args_again();
  if (z.counters) zero_rows<D>(z);
}

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
      if (row < rows) write_rows<D, NT>(args, seg, r, nt, row, slot, padded, sum);
    }
  }
}

template <int D, int NT>
int launch_many(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.nwg + 7) / 8 * 8)), threads(kThreads);
  hipLaunchKernelGGL((attend_many_kernel<D, NT>), grid, threads, 0, st, a);
  if (const int e = launch_status()) return e;
  return launch_join_many<D, NT, ManyDeal>(a, st);
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
  return launch_join_few<D, FewDeal>(a, st);
}

}  // namespace
}  // namespace umic

extern "C" int64_t umic_cache_attention_workspace_bytes(int64_t S, int64_t Hq, int64_t Hk,
                                                        int64_t D) {
  return umic::workspace_bytes(S, Hq, Hk, D, umic::few_of(D));
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
  const AttnCall call = {q,    k,    v,    out,    table,      kv_lens,  q_lens,  B,      S,
                         Hq,   Hk,   D,    q_sb,   q_ss,       q_sh,     o_sb,    o_ss,   o_sh,
                         c_sb, c_sh, c_ss, blocks, block_rows, table_ld, table_w, kv_len, causal,
                         scale, counters, workspace, workspace_bytes};
  AttnArgs a = {};
  Shape s;
  if (const int e = attn_args(call, 8, few_of(D), a, s)) return e == 1 ? UMIC_OK : e;
  // Single tokens of a few segments, up to a quarter of the CUs': a workgroup to a
  // CU.  The second hides the starts and ends of segments; with few it only doubles
  // their parts (8 segments of 12288 keys 18 us for 25, 64 of 1024 14.5 for 15.4; 128
  // of 300 15.2 for 13.6, 64 ragged requests 74 for 60).
  const int cus = s.nwg / few_of(D);
  if (s.nt == 0 && B * Hk * 4 <= cus) a.nwg = a.some = cus;
  hipStream_t st = as_stream(stream);
  if (D == 64) return launch<64>(s, a, st);
  if (D == 128) return launch<128>(s, a, st);
  return launch<256>(s, a, st);
}
