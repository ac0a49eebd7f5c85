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
// Nothing goes through LDS until the four waves of a workgroup, which take 32
// keys each of a tile of 128, are joined.
//
// The tiles of all requests, in one row, are dealt evenly over the launch's
// workgroups, so requests of all lengths fill the chip alike.  A workgroup that
// has a part of a request's tiles leaves (max, sum, output) in the workspace: at
// most two such parts each, the first and the last of its tiles; a second kernel
// joins the parts in a fixed order.
//
// p is split in two bf16 parts (p = hi + lo to 2^-17), each its own product: one
// rounding to bf16 would weigh as much as the output's own.
#include "common.hpp"
#include "gemm_ks.hpp"  // device_cus

namespace umic {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kStep = 32;              // keys of a wave's step
constexpr int kTile = kStep * kWaves;  // keys of a workgroup's step

struct AttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  const int32_t* table;   // or NULL: request b is block b
  const int32_t* kv_len;  // or NULL: len
  const int32_t* q_len;   // or NULL: S
  float* part;            // [2 nwg][16 NT][D + 2]
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss, c_sb, c_sh, c_ss, table_ld;
  int64_t cap;            // keys a request can hold
  int B, S, Hk, G, rb;    // rb: row blocks of a (request, key head)
  int len, blocks, shift, causal, nwg;
  float c;                // scale * log2(e)
};

__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  const int n = a.kv_len ? a.kv_len[b] : a.len;
  return n < 0 ? 0 : (int64_t)n > a.cap ? (int)a.cap : n;
}

__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) {
  return (keys_of(a, b) + kTile - 1) / kTile;
}

__device__ __forceinline__ int new_of(const AttnArgs& a, int b) {
  const int n = a.q_len ? a.q_len[b] : a.S;
  return n < 0 ? 0 : n > a.S ? a.S : n;
}

// Sum of one value per thread of the workgroup.
__device__ __forceinline__ int block_sum(int v, int* sums) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v += __shfl_xor(v, m, kWave);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sums[threadIdx.x / kWave] = v;
  __syncthreads();
  return sums[0] + sums[1] + sums[2] + sums[3];
}

// Tiles of the requests before b, and of all.
__device__ __forceinline__ void tiles_before(const AttnArgs& a, int b, int* sums, int64_t& before,
                                             int64_t& all) {
  if (!a.kv_len) {
    const int64_t n = tiles_of(a, 0);
    before = n * b;
    all = n * a.B;
    return;
  }
  int x = 0, y = 0;
  for (int i = threadIdx.x; i < a.B; i += kThreads) {
    const int n = tiles_of(a, i);
    y += n;
    if (i < b) x += n;
  }
  before = block_sum(x, sums);
  all = block_sum(y, sums);
}

// The request that holds tile t of all (t < all), and the tiles before it.
__device__ __forceinline__ int request_at(const AttnArgs& a, int64_t t, int* sums, int* found,
                                          int64_t& before) {
  if (!a.kv_len) {
    const int n = tiles_of(a, 0);
    const int b = (int)(t / n);
    before = (int64_t)b * n;
    return b;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int carry = 0;
  for (int base = 0;; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    const int n = i < a.B ? tiles_of(a, i) : 0;
    int x = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int y = __shfl_up(x, d, kWave);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == kWave - 1) sums[wave] = x;
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    x += carry;
    for (int w = 0; w < wave; ++w) x += sums[w];
    if (t >= x - n && t < x) {
      found[0] = i;
      found[1] = x - n;
    }
    carry += sums[0] + sums[1] + sums[2] + sums[3];
    __syncthreads();
    if (found[0] >= 0 || base + kThreads >= a.B) break;
  }
  before = found[1];
  return found[0];
}

__device__ __forceinline__ bf16x8_t as_bf(const u32x4& v) { return __builtin_bit_cast(bf16x8_t, v); }

// The low (hi: high) halves of two words side by side.
__device__ __forceinline__ uint32_t pair_lo(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t pair_hi(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Rows of the output that one workgroup's (or the join's) result goes to.
struct RowOf {
  int s, g;
};

template <int D, int NT>
__global__ __launch_bounds__(kThreads) void cache_attention_kernel(AttnArgs a) {
  constexpr int KK = D / 32;  // 32-wide steps of a score's product
  constexpr int DV = D / 16;  // output columns of a lane, V columns it reads
  constexpr int VW = DV / 2;  // 32-bit words of those
  constexpr int LDR = D + 4;  // row of the join's LDS, in floats
  __shared__ int sums[kWaves];
  __shared__ int found[2];
  __shared__ float ml[kWaves][NT * 16][2];
  __shared__ float acc_lds[kWaves][16][LDR];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;

  const int per = a.Hk * a.rb;  // (key head, row block) pairs of a request
  int64_t before, all;
  tiles_before(a, 0, sums, before, all);
  const int64_t units = all * per;
  const int64_t wg = blockIdx.x;
  const int64_t nwg = units < a.nwg ? units : a.nwg;  // each has a tile
  if (wg >= nwg) return;
  int64_t u = wg * units / nwg;
  const int64_t u_end = (wg + 1) * units / nwg;
  int b = request_at(a, u / per, sums, found, before);
  b = __builtin_amdgcn_readfirstlane(b);

  while (u < u_end) {
    const int len = __builtin_amdgcn_readfirstlane(keys_of(a, b));
    const int tiles = (len + kTile - 1) / kTile;
    if (tiles == 0) {
      ++b;
      continue;
    }
    const int64_t in = u - before * per;  // unit of this request
    const int pair = (int)(in / tiles);
    const int t0 = (int)(in - (int64_t)pair * tiles);
    const int t1 = (int)(tiles - t0 < u_end - u ? tiles : t0 + (u_end - u));
    const int h = pair / a.rb, rb = pair - h * a.rb;
    const int fresh = __builtin_amdgcn_readfirstlane(new_of(a, b));

    // this lane's rows: row r is head g of new token s
    int lim[NT];
    u32x4 qf[NT][KK];
    const int rows = a.S * a.G;
    const int r0 = rb * 16 * NT;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int r = r0 + nt * 16 + n16;
      if (r >= rows) r = rows - 1;  // computed again, not written
      const int s = r / a.G, g = r - s * a.G;
      lim[nt] = a.causal ? min(len, len - fresh + s + 1) : len;
      const uint16_t* qp = a.q + b * a.q_sb + (int64_t)(h * a.G + g) * a.q_sh + s * a.q_ss + g4 * 8;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[nt][kk] = *reinterpret_cast<const u32x4*>(qp + kk * 32);
    }
    // keys below lo are seen by all rows, keys from hi on by none
    const int r1 = min(rows, r0 + 16 * NT) - 1;
    const int lo = a.causal ? min(len, len - fresh + r0 / a.G + 1) : len;
    const int hi = a.causal ? min(len, len - fresh + r1 / a.G + 1) : len;

    float m[NT], l[NT];
    f32x4_t acc[NT][DV];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -__builtin_inff();
      l[nt] = 0.0f;
#pragma unroll
      for (int e = 0; e < DV; ++e) acc[nt][e] = f32x4_t{0, 0, 0, 0};
    }

    for (int t = t0; t < t1; ++t) {
      const int k0 = t * kTile + wave * kStep;
      if (k0 >= hi) break;
      // where the two key tiles of 16 lie: a page never ends inside one
      const uint16_t* kb[2];
      const uint16_t* vb[2];
      int row0[2];
      bool ok[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = k0 + 16 * i;
        ok[i] = key < len;
        int64_t block = b;
        row0[i] = ok[i] ? key : 0;
        if (a.table) {
          const int at = row0[i] >> a.shift;
          const int page = a.table[(int64_t)b * a.table_ld + at];
          ok[i] = ok[i] && page >= 0 && page < a.blocks;  // a page outside the pool: not seen
          block = ok[i] ? page : 0;
          row0[i] -= at << a.shift;
        }
        const int64_t off = block * a.c_sb + h * a.c_sh;
        kb[i] = a.k + off;
        vb[i] = a.v + off;
      }
      const bool edge = k0 + kStep > lo || !ok[0] || !ok[1];
      u32x4 kf[2][KK];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // rows past the length are read again from a row that is there
        const int key = k0 + 16 * i + n16;
        const int row = key < len && ok[i] ? row0[i] + n16 : row0[i];
        const uint16_t* p = kb[i] + row * a.c_ss + g4 * 8;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) kf[i][kk] = *reinterpret_cast<const u32x4*>(p + kk * 32);
      }
      uint32_t vr[8][VW];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = j >> 2, at = 4 * g4 + (j & 3);
        const bool there = k0 + 16 * i + at < len && ok[i];
        const uint32_t* p = reinterpret_cast<const uint32_t*>(
            vb[i] + (row0[i] + (there ? at : 0)) * a.c_ss + n16 * DV);
#pragma unroll
        for (int w = 0; w < VW; ++w) vr[j][w] = p[w];
        if (edge && !there)  // 0 * inf is not 0
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[j][w] = 0;
      }
      f32x4_t sc[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc[nt][i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            sc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(kf[i][kk]), as_bf(qf[nt][kk]),
                                                                 sc[nt][i], 0, 0, 0);
        }
      u32x4 ph[NT], pl[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = sc[nt][j >> 2][j & 3] * a.c;
          if (edge) {
            const int key = k0 + 16 * (j >> 2) + 4 * g4 + (j & 3);
            if (key >= lim[nt] || !ok[j >> 2]) x[j] = -__builtin_inff();
          }
        }
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x[j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        const float mn = fmaxf(m[nt], mx);
        const float base = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m[nt] - base);
        m[nt] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = __builtin_amdgcn_exp2f(x[j] - base);
          sum += x[j];
        }
        l[nt] = l[nt] * al + sum;
#pragma unroll
        for (int e = 0; e < DV; ++e) acc[nt][e] *= al;
        ph[nt] = pack8(x);
        float y[8];
        unpack8(ph[nt], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[j] - y[j];
        pl[nt] = pack8(y);
      }
      // Where some rows do not see some of these keys, p = 0 has to hide a v that is
      // not finite, and 0 * inf is not 0: such elements leave the product, and the rows
      // that see them get theirs one by one.
      if (edge && a.causal && hi > lo) {
        bool wild = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const uint32_t x = vr[j][w];
            const bool l16 = (x & 0x7f80u) == 0x7f80u, h16 = (x & 0x7f800000u) == 0x7f800000u;
            wild |= l16 | h16;
            vr[j][w] = x & ~((l16 ? 0xffffu : 0u) | (h16 ? 0xffff0000u : 0u));
          }
        if (__any(wild)) {
#pragma unroll 1
          for (int key = 0; key < kStep; ++key) {
            const int i = key >> 4, at = key & 15, j = i * 4 + (at & 3);
            if (k0 + key >= len || !(i ? ok[1] : ok[0])) continue;
            const uint16_t* vp = (i ? vb[1] : vb[0]) + ((i ? row0[1] : row0[0]) + at) * a.c_ss;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t wh = ph[nt][0], wl = pl[nt][0];
#pragma unroll
              for (int y = 1; y < 4; ++y) {
                wh = (j >> 1) == y ? ph[nt][y] : wh;
                wl = (j >> 1) == y ? pl[nt][y] : wl;
              }
              float p = (j & 1) ? bf_hi(wh) + bf_hi(wl) : bf_lo(wh) + bf_lo(wl);
              p = __shfl(p, n16 + 16 * (at >> 2), kWave);
              if (k0 + key < lim[nt])
#pragma unroll
                for (int e = 0; e < DV; ++e)
#pragma unroll
                  for (int y = 0; y < 4; ++y) {
                    const float x = bf2f(vp[(4 * g4 + y) * DV + e]);
                    if (!(__builtin_fabsf(x) < __builtin_inff())) acc[nt][e][y] += p * x;
                  }
            }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        u32x4 v0, v1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v0[j] = pair_lo(vr[2 * j][w], vr[2 * j + 1][w]);
          v1[j] = pair_hi(vr[2 * j][w], vr[2 * j + 1][w]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          f32x4_t& c0 = acc[nt][2 * w];
          f32x4_t& c1 = acc[nt][2 * w + 1];
          c0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v0), as_bf(ph[nt]), c0, 0, 0, 0);
          c1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v1), as_bf(ph[nt]), c1, 0, 0, 0);
          c0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v0), as_bf(pl[nt]), c0, 0, 0, 0);
          c1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf(v1), as_bf(pl[nt]), c1, 0, 0, 0);
        }
      }
    }

    // join the waves
    const bool whole = t0 == 0 && t1 == tiles;
    const int slot = (int)wg * 2 + (t0 == 0 ? 1 : 0);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += __shfl_xor(l[nt], 16, kWave);
      l[nt] += __shfl_xor(l[nt], 32, kWave);
      if (g4 == 0) {
        ml[wave][nt * 16 + n16][0] = m[nt];
        ml[wave][nt * 16 + n16][1] = l[nt];
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DV; ++e) acc_lds[wave][n16][(4 * g4 + i) * DV + e] = acc[nt][e][i];
      __syncthreads();
      // thread: row tid / 16, columns DV (tid % 16) ..
      const int rr = threadIdx.x >> 4, col = (threadIdx.x & 15) * DV;
      const int r = r0 + nt * 16 + rr;
      if (r < rows) {
        float mx = ml[0][nt * 16 + rr][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, ml[w][nt * 16 + rr][0]);
        const float base = mx == -__builtin_inff() ? 0.0f : mx;
        float o[DV] = {};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(ml[w][nt * 16 + rr][0] - base);
          sum += ml[w][nt * 16 + rr][1] * f;
#pragma unroll
          for (int e = 0; e < DV; ++e) o[e] += acc_lds[w][rr][col + e] * f;
        }
        if (whole) {
          const int s = r / a.G, g = r - s * a.G;
          const float inv = s < fresh && sum != 0.0f ? 1.0f / sum : 0.0f;
          uint16_t* op = a.out + b * a.o_sb + s * a.o_ss + (int64_t)(h * a.G + g) * a.o_sh + col;
#pragma unroll
          for (int e = 0; e < DV; ++e) op[e] = (uint16_t)f2bf(inv == 0.0f ? 0.0f : o[e] * inv);
        } else {
          float* p = a.part + ((int64_t)slot * 16 * NT + nt * 16 + rr) * (D + 2);
#pragma unroll
          for (int e = 0; e < DV; ++e) p[col + e] = o[e];
          if (col == 0) {
            p[D] = mx;
            p[D + 1] = sum;
          }
        }
      }
    }

    u += t1 - t0;
    if (u - before * per >= (int64_t)tiles * per) {
      before += tiles;
      ++b;
    }
  }
}

// Joins the parts of one (request, key head, row block), in the order of its
// keys; rows without a key become zero.
template <int D, int NT>
__global__ __launch_bounds__(kThreads) void cache_attention_join_kernel(AttnArgs a) {
  __shared__ int sums[kWaves];
  const int per = a.Hk * a.rb;
  const int b = blockIdx.x / per, pair = blockIdx.x - b * per;
  const int h = pair / a.rb, rb = pair - h * a.rb;
  int64_t before, all;
  tiles_before(a, b, sums, before, all);
  const int tiles = tiles_of(a, b);
  const int64_t units = all * per;
  const int64_t first = before * per + (int64_t)pair * tiles;
  int64_t w0 = 0, w1 = -1;  // the workgroups that hold its tiles
  if (tiles) {
    const int64_t nwg = units < a.nwg ? units : a.nwg;
    w0 = ((first + 1) * nwg - 1) / units;
    w1 = ((first + tiles) * nwg - 1) / units;
    if (w0 == w1) return;
  }
  const int fresh = new_of(a, b);
  const int rows = min(a.S * a.G - rb * 16 * NT, 16 * NT);
  for (int i = threadIdx.x; i < rows * D; i += kThreads) {
    const int rr = i / D, col = i - rr * D;
    const int r = rb * 16 * NT + rr, s = r / a.G, g = r - s * a.G;
    float mx = -__builtin_inff();
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t slot = w * 2 + (w == w0 ? 1 : 0);
      mx = fmaxf(mx, a.part[(slot * 16 * NT + rr) * (D + 2) + D]);
    }
    const float base = mx == -__builtin_inff() ? 0.0f : mx;
    float o = 0.0f, sum = 0.0f;
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t slot = w * 2 + (w == w0 ? 1 : 0);
      const float* p = a.part + (slot * 16 * NT + rr) * (D + 2);
      const float f = __builtin_amdgcn_exp2f(p[D] - base);
      o += p[col] * f;
      sum += p[D + 1] * f;
    }
    const bool none = s >= fresh || sum == 0.0f;
    a.out[b * a.o_sb + s * a.o_ss + (int64_t)(h * a.G + g) * a.o_sh + col] =
        (uint16_t)f2bf(none ? 0.0f : o / sum);
  }
}

struct Shape {
  int nt, rb, nwg;
};

// Row tiles of a workgroup, row blocks, workgroups.
Shape shape_of(int64_t rows, int64_t D, int64_t cus) {
  Shape s;
  s.nt = rows <= 16 ? 1 : rows <= 32 || D > 128 ? 2 : 4;
  s.rb = (int)((rows + 16 * s.nt - 1) / (16 * s.nt));
  s.nwg = (int)(cus * (s.nt == 1 ? 2 : 1));
  return s;
}

template <int D, int NT>
int launch(const AttnArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((cache_attention_kernel<D, NT>), dim3((unsigned)a.nwg), dim3(kThreads), 0, st,
                     a);
  if (int e = launch_status()) return e;
  hipLaunchKernelGGL((cache_attention_join_kernel<D, NT>), dim3((unsigned)(a.B * a.Hk * a.rb)),
                     dim3(kThreads), 0, st, a);
  return launch_status();
}

template <int D>
int launch_nt(int nt, const AttnArgs& a, hipStream_t st) {
  if (nt == 1) return launch<D, 1>(a, st);
  if constexpr (D <= 128)
    if (nt == 4) return launch<D, 4>(a, st);
  return launch<D, 2>(a, st);
}

bool head_dim_ok(int64_t D) { return D == 64 || D == 128 || D == 256; }

}  // namespace
}  // namespace umic

extern "C" int64_t umic_cache_attention_workspace_bytes(int64_t S, int64_t Hq, int64_t Hk,
                                                        int64_t D) {
  using namespace umic;
  if (S <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || !head_dim_ok(D) || S > (1 << 20) || Hq > (1 << 16))
    return 0;
  const Shape s = shape_of(S * (Hq / Hk), D, device_cus());
  return (int64_t)s.nwg * 2 * 16 * s.nt * (D + 2) * 4;
}

extern "C" int umic_cache_attention_bf16(
    const void* q, const void* k, const void* v, void* out, const int32_t* table,
    const int32_t* kv_lens, const int32_t* q_lens, int64_t B, int64_t S, int64_t Hq, int64_t Hk,
    int64_t D, int64_t q_sb, int64_t q_ss, int64_t q_sh, int64_t o_sb, int64_t o_ss, int64_t o_sh,
    int64_t c_sb, int64_t c_sh, int64_t c_ss, int64_t blocks, int64_t block_rows, int64_t table_ld,
    int64_t table_w, int64_t kv_len, int causal, float scale, void* workspace,
    int64_t workspace_bytes, void* stream) {
  using namespace umic;
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || blocks < 0 || block_rows < 0 ||
      workspace_bytes < 0)
    return UMIC_ERR_INVALID_ARG;
  if (B == 0 || S == 0 || Hq == 0) return UMIC_OK;
  if (Hk == 0 || Hq % Hk) return UMIC_ERR_INVALID_ARG;
  if (!q || !out || !workspace) return UMIC_ERR_INVALID_ARG;
  if (!head_dim_ok(D)) return UMIC_ERR_UNSUPPORTED;
  int64_t cap = block_rows;
  int shift = 0;
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
  if (B > (1 << 20) || S > (1 << 20) || Hq > (1 << 16) || cap > ((int64_t)1 << 30) ||
      blocks > ((int64_t)1 << 30))
    return UMIC_ERR_UNSUPPORTED;
  const Shape s = shape_of(S * G, D, cus);
  if (workspace_bytes < (int64_t)s.nwg * 2 * 16 * s.nt * (D + 2) * 4) return UMIC_ERR_INVALID_ARG;
  // tiles of all requests, and joins, are counted in 32 bits
  if (B * ((cap + kTile - 1) / kTile) > 0x7fffffff || B * Hk * s.rb > 0x7fffffff)
    return UMIC_ERR_UNSUPPORTED;
  AttnArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.out = (uint16_t*)out, a.table = table, a.kv_len = kv_lens, a.q_len = q_lens;
  a.part = (float*)workspace;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.o_sb = o_sb, a.o_ss = o_ss, a.o_sh = o_sh;
  a.c_sb = c_sb, a.c_sh = c_sh, a.c_ss = c_ss, a.table_ld = table_ld, a.cap = cap;
  a.B = (int)B, a.S = (int)S, a.Hk = (int)Hk, a.G = (int)G, a.rb = s.rb;
  a.len = kv_lens ? 0 : (int)kv_len, a.blocks = (int)blocks, a.shift = shift;
  a.causal = causal != 0, a.nwg = s.nwg, a.c = scale * 1.4426950408889634f;
  hipStream_t st = as_stream(stream);
  if (D == 64) return launch_nt<64>(s.nt, a, st);
  if (D == 128) return launch_nt<128>(s.nt, a, st);
  return launch_nt<256>(s.nt, a, st);
}
