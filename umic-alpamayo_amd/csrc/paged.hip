// Pages of a shared key / value pool: block tables and slot maps from request
// lengths, wholly on the device.
//
// A pool of P pages of `page` tokens each is shared by R requests.  table[r]
// names the pages of request r in order, ring holds the free ones as a queue
// (cursor = head, count), kv_len[r] counts its tokens.  One call is one step:
// request r keeps its first kept = clamp(keep[r], 0, kv_len[r]) tokens and gets
// new[r] more.  With have = ceil(kv_len / page) and need = ceil((kept + new) /
// page), pages [need, have) of its row go to the queue's tail and pages [have,
// need) come from its head, in request order; token i lies at position p = kept
// + i, in slot table[r][p / page] * page + p % page.
//
// Latency: a step of eight requests moves a few hundred bytes.  The prefix sums
// over requests are what has to be waited for.
#include "common.hpp"

namespace umic {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

struct PlanArgs {
  const int32_t* kv_len;
  const int32_t* fresh;  // new tokens
  const int32_t* keep;   // or NULL: all
  const int32_t* delta;  // or NULL: 0
  int32_t* table;
  int32_t* ring;
  const int32_t* cursor;
  int32_t* kv_out;
  int32_t* cursor_out;
  int32_t* starts;
  int64_t* slots;
  int64_t* positions;
  int64_t ld, tokens, row;
  int R, W, P, shift;
};

struct Request {
  int kept, have, need, fresh;
  bool bad_state, too_long;
};

__device__ __forceinline__ Request request_of(const PlanArgs& a, int r) {
  const int page = 1 << a.shift;
  const int len = a.kv_len[r];
  const int k = a.keep ? a.keep[r] : len;
  Request q;
  q.kept = max(0, min(k, len));
  q.fresh = max(0, a.fresh[r]);
  const int64_t after = (int64_t)q.kept + q.fresh;
  q.bad_state = len < 0 || (int64_t)len > ((int64_t)a.W << a.shift);
  q.too_long = after > ((int64_t)a.W << a.shift);
  q.have = q.bad_state ? 0 : (int)(((int64_t)len + page - 1) >> a.shift);
  q.need = q.too_long ? 0 : (int)((after + page - 1) >> a.shift);
  return q;
}

// Sums of one value per thread: exclusive prefix over the block, and the total.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  __syncthreads();  // sums may still be read from the call before
  if (lane == kWave - 1) sums[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before + x - v;
}

// One workgroup: the sums over requests, the refusals, the pages that move, the
// new lengths.  A refused step changes nothing: lengths and queue as they were,
// no tokens, every slot -1, the reason in cursor_out[3].
__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(PlanArgs a) {
  __shared__ int64_t sums[kPlanWaves];
  const int tid = threadIdx.x;
  const int head = a.cursor[0], free = a.cursor[1];
  int64_t gave = 0, took = 0, fresh = 0, bad = 0, lng = 0, wide = 0;
  for (int r = tid; r < a.R; r += kPlanThreads) {
    const Request q = request_of(a, r);
    gave += max(0, q.have - q.need);
    took += max(0, q.need - q.have);
    fresh += q.fresh;
    bad |= q.bad_state;
    lng |= q.too_long;
    wide |= a.row > 0 && q.fresh > a.row;
  }
  int64_t gave_all, took_all, fresh_all, flags;
  block_scan(gave, sums, gave_all);
  block_scan(took, sums, took_all);
  block_scan(fresh, sums, fresh_all);
  block_scan(bad | lng << 20 | wide << 40, sums, flags);
  int status = UMIC_PLAN_OK;
  if ((flags & 0xfffff) || head < 0 || head >= a.P || free < 0 || free > a.P ||
      free + gave_all > a.P)
    status = UMIC_PLAN_BAD_STATE;
  else if ((flags >> 20) & 0xfffff)
    status = UMIC_PLAN_TOO_LONG;
  else if ((flags >> 40) || (a.row <= 0 && fresh_all > a.tokens))
    status = UMIC_PLAN_NO_ROOM;
  else if (took_all > free + gave_all)
    status = UMIC_PLAN_NO_PAGES;

  // pages given back, then pages taken: one wave to a request
  for (int phase = 0; phase < 2; ++phase) {
    int64_t carry = 0;
    for (int base = 0; base < a.R; base += kPlanThreads) {
      __shared__ int from[kPlanThreads], count[kPlanThreads];
      __shared__ int64_t at[kPlanThreads];
      const int r = base + tid;
      Request q = {};
      if (r < a.R) q = request_of(a, r);
      const int n = phase ? max(0, q.need - q.have) : max(0, q.have - q.need);
      int64_t total, before = block_scan(n, sums, total);
      from[tid] = phase ? q.have : q.need;
      count[tid] = status ? 0 : n;
      at[tid] = carry + before;
      __syncthreads();
      const int here = min(kPlanThreads, a.R - base);
      for (int j = tid / kWave; j < here; j += kPlanWaves) {
        int32_t* row = a.table + (int64_t)(base + j) * a.ld + from[j];
        for (int w = tid & (kWave - 1); w < count[j]; w += kWave) {
          const int64_t i = (int64_t)head + (phase ? 0 : free) + at[j] + w;
          int32_t* cell = a.ring + i % a.P;
          if (phase)
            row[w] = *cell;
          else
            *cell = row[w];
        }
      }
      carry += total;
      __syncthreads();
    }
  }

  // lengths and starts last: kv_out may be kv_len
  int64_t carry = 0;
  for (int base = 0; base < a.R; base += kPlanThreads) {
    const int r = base + tid;
    Request q = {};
    if (r < a.R) q = request_of(a, r);
    int64_t total, before = block_scan(q.fresh, sums, total);
    if (r < a.R) {
      a.starts[r] = status ? 0 : (int32_t)(carry + before);
      a.kv_out[r] = status ? a.kv_len[r] : q.kept + q.fresh;
    }
    carry += total;
  }
  if (tid == 0) {
    a.starts[a.R] = status ? 0 : (int32_t)fresh_all;
    a.cursor_out[0] = status ? head : (int)((head + took_all) % a.P);
    a.cursor_out[1] = status ? free : (int)(free + gave_all - took_all);
    a.cursor_out[2] = status ? 0 : (int)fresh_all;
    a.cursor_out[3] = status;
  }
}

// A token's slot and position, from what the plan has written.
__global__ __launch_bounds__(256) void slot_map_kernel(PlanArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  int r;
  int64_t i;
  bool real;
  if (a.row > 0) {
    r = (int)(t / a.row);
    i = t - (int64_t)r * a.row;
    real = i < a.starts[r + 1] - a.starts[r];
  } else {
    int lo = 0, hi = a.R;  // starts[lo] <= t < starts[hi], if there is such a request
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] <= t) lo = mid; else hi = mid;
    }
    r = lo;
    i = t - a.starts[r];
    real = t < a.starts[a.R];
  }
  int64_t slot = -1, position = 0;
  if (real) {
    const int64_t p = a.kv_out[r] - (a.starts[r + 1] - a.starts[r]) + i;
    slot = ((int64_t)a.table[(int64_t)r * a.ld + (p >> a.shift)] << a.shift) +
           (p & ((1 << a.shift) - 1));
    position = p + (a.delta ? a.delta[r] : 0);
  }
  a.slots[t] = slot;
  a.positions[t] = position;
}

}  // namespace
}  // namespace umic

extern "C" int umic_page_plan(const int32_t* kv_len, const int32_t* new_len, const int32_t* keep,
                              const int32_t* delta, int32_t* table, int32_t* ring,
                              const int32_t* cursor, int32_t* kv_len_out, int32_t* cursor_out,
                              int32_t* starts, int64_t* slots, int64_t* positions, int64_t R,
                              int64_t W, int64_t table_ld, int64_t pages, int64_t page_size,
                              int64_t tokens, int64_t row, void* stream) {
  using namespace umic;
  if (R < 0 || W < 0 || pages < 0 || tokens < 0 || row < 0 || page_size <= 0)
    return UMIC_ERR_INVALID_ARG;
  if (R == 0) return tokens ? UMIC_ERR_INVALID_ARG : UMIC_OK;
  if (W == 0 || pages == 0 || table_ld < W) return UMIC_ERR_INVALID_ARG;
  if (row > 0 && (tokens % row || tokens / row != R)) return UMIC_ERR_INVALID_ARG;
  if (!kv_len || !new_len || !table || !ring || !cursor || !kv_len_out || !cursor_out ||
      !starts || (tokens && (!slots || !positions)))
    return UMIC_ERR_INVALID_ARG;
  if (page_size < 16 || (page_size & (page_size - 1))) return UMIC_ERR_UNSUPPORTED;
  constexpr int64_t kMost = (int64_t)1 << 30;
  if (R > kMost || W > kMost || pages > kMost || tokens > kMost || page_size > kMost)
    return UMIC_ERR_UNSUPPORTED;
  PlanArgs a = {kv_len, new_len, keep, delta, table, ring, cursor, kv_len_out, cursor_out,
                starts, slots, positions, table_ld, tokens, row, (int)R, (int)W, (int)pages,
                __builtin_ctzll((unsigned long long)page_size)};
  hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(page_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  if (int e = launch_status()) return e;
  if (tokens == 0) return UMIC_OK;
  hipLaunchKernelGGL(slot_map_kernel, dim3((unsigned)((tokens + 255) / 256)), dim3(256), 0, st, a);
  return launch_status();
}
