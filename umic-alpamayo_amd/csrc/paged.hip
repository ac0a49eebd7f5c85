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
// Latency: a step of eight requests moves a few hundred bytes.  One workgroup does
// all that depends on the sums over requests, with one scan of all of them at once
// for up to kPlanThreads requests, and the slots of up to kSlotsHere tokens; more
// tokens' slots are a second launch's.  8 requests' tokens 3.5 us, a launch being 2.3;
// 256 requests, half of them anew, with 34816 slots 7 and 4.
#include "common.hpp"

namespace umic {
namespace {

// A workgroup of 256 threads for up to as many requests, else of 1024: its barriers
// are what a small step waits for.
constexpr int kFewRequests = 256;
constexpr int kPlanThreads = 1024;
constexpr int kSlotsHere = 2048;

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

// What a step does to one request.
struct Request {
  int kept, have, need, fresh, bad;  // bad: 1 its state is out of range, 2 too long
  __device__ __forceinline__ int gives() const { return max(0, have - need); }
  __device__ __forceinline__ int takes() const { return max(0, need - have); }
};

__device__ __forceinline__ Request request_of(const PlanArgs& a, int r) {
  Request q = {};
  if (r >= a.R) return q;
  const int64_t row = (int64_t)a.W << a.shift;
  const int64_t most = row < 0x7fffffff ? row : 0x7fffffff;  // lengths are 32-bit
  const int len = a.kv_len[r];
  q.kept = max(0, min(a.keep ? a.keep[r] : len, len));
  q.fresh = max(0, a.fresh[r]);
  const int64_t after = (int64_t)q.kept + q.fresh;
  const int64_t up = ((int64_t)1 << a.shift) - 1;
  if (len < 0 || len > most)
    q.bad = 1;
  else
    q.have = (int)((len + up) >> a.shift);
  if (after > most)
    q.bad |= 2;
  else
    q.need = (int)((after + up) >> a.shift);
  return q;
}

struct Sums {
  int64_t gives, takes, fresh;
};

// Sums over the requests before this thread's, and over all; `bad` of all.
template <int THREADS>
__device__ __forceinline__ Sums scan(const Request& q, int64_t row, Sums& all, int& bad,
                                     Sums (&part)[THREADS / kWave], int (&flag)[THREADS / kWave]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  Sums x = {q.gives(), q.takes(), q.fresh};
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t g = __shfl_up(x.gives, d, kWave), t = __shfl_up(x.takes, d, kWave),
                  f = __shfl_up(x.fresh, d, kWave);
    if (lane >= d) x.gives += g, x.takes += t, x.fresh += f;
  }
  const int what = q.bad | (row > 0 && q.fresh > row ? 4 : 0);
  const int any = (__any(what & 1) ? 1 : 0) | (__any(what & 2) ? 2 : 0) | (__any(what & 4) ? 4 : 0);
  __syncthreads();  // part may still be read from the call before
  if (lane == kWave - 1) part[wave] = x;
  if (lane == 0) flag[wave] = any;
  __syncthreads();
  Sums before = {x.gives - q.gives(), x.takes - q.takes(), x.fresh - q.fresh};
  all = {0, 0, 0};
  bad = 0;
#pragma unroll 2
  for (int w = 0; w < THREADS / kWave; ++w) {
    const Sums p = part[w];
    if (w < wave) before.gives += p.gives, before.takes += p.takes, before.fresh += p.fresh;
    all.gives += p.gives, all.takes += p.takes, all.fresh += p.fresh;
    bad |= flag[w];
  }
  return before;
}

// Token t's slot and position, from what the plan has written; starts(r): the
// tokens of the requests before r, fresh ones; len(r): its length after the step.
template <typename Starts, typename Len>
__device__ __forceinline__ void map_slot(const PlanArgs& a, int64_t t, Starts starts, Len len) {
  int r;
  int64_t i;
  if (a.row > 0) {
    r = (int)(t / a.row);
    i = t - (int64_t)r * a.row;
  } else {
    int lo = 0, hi = a.R;  // starts[lo] <= t < starts[hi], if there is such a request
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts(mid) <= t) lo = mid; else hi = mid;
    }
    r = lo;
    i = t - starts(r);
  }
  const int64_t n = starts(r + 1) - starts(r);
  int64_t slot = -1, position = 0;
  if (i < n) {
    const int64_t p = len(r) - n + i;
    slot = ((int64_t)a.table[(int64_t)r * a.ld + (p >> a.shift)] << a.shift) +
           (p & (((int64_t)1 << a.shift) - 1));
    position = p + (a.delta ? a.delta[r] : 0);
  }
  a.slots[t] = slot;
  a.positions[t] = position;
}

// The sums over requests, the refusals, the pages that move, the new lengths.  A
// refused step changes nothing: lengths and queue as they were, no tokens, every
// slot -1, the reason in cursor_out[3].
template <int THREADS>
__global__ __launch_bounds__(THREADS) void page_plan_kernel(PlanArgs a) {
  __shared__ Sums part[THREADS / kWave];
  __shared__ int flag[THREADS / kWave];
  __shared__ int from[THREADS], at[THREADS];
  __shared__ int starts[THREADS + 1], lens[THREADS];
  const int tid = threadIdx.x;
  const int head = a.cursor[0], free = a.cursor[1];
  const bool once = a.R <= THREADS;
  const Request mine = request_of(a, tid);
  Sums all;
  int bad;
  Sums before = scan<THREADS>(mine, a.row, all, bad, part, flag);
  for (int base = THREADS; base < a.R; base += THREADS) {
    Sums more;
    int b;
    scan<THREADS>(request_of(a, base + tid), a.row, more, b, part, flag);
    all.gives += more.gives, all.takes += more.takes, all.fresh += more.fresh;
    bad |= b;
  }
  int status = UMIC_PLAN_OK;
  if ((bad & 1) || head < 0 || head >= a.P || free < 0 || free > a.P || free + all.gives > a.P)
    status = UMIC_PLAN_BAD_STATE;
  else if (bad & 2)
    status = UMIC_PLAN_TOO_LONG;
  else if ((bad & 4) || (a.row <= 0 && all.fresh > a.tokens))
    status = UMIC_PLAN_NO_ROOM;
  else if (all.takes > free + all.gives)
    status = UMIC_PLAN_NO_PAGES;

  // pages given back, then pages taken
  for (int phase = 0; phase < 2; ++phase) {
    if (status || (phase ? all.takes : all.gives) == 0) continue;
    int64_t carry = 0;
    for (int base = 0; base < a.R; base += THREADS) {
      Request q = mine;
      Sums b = before, more;
      if (!once) {
        int f;
        q = request_of(a, base + tid);
        b = scan<THREADS>(q, a.row, more, f, part, flag);
      }
      // pages below P, as the step was not refused
      from[tid] = phase ? q.have : q.need;
      at[tid] = (int)(phase ? b.takes : b.gives);
      __syncthreads();
      const int here = min(THREADS, a.R - base);
      const int total = (int)(once ? (phase ? all.takes : all.gives)
                                   : (phase ? more.takes : more.gives));
      for (int k = tid; k < total; k += THREADS) {
        int j = 0;  // the last request with at <= k
        for (int hi = here; hi - j > 1;) {
          const int mid = (j + hi) >> 1;
          if (at[mid] <= k) j = mid; else hi = mid;
        }
        int32_t* cell = a.table + (int64_t)(base + j) * a.ld + from[j] + (k - at[j]);
        int64_t i = (int64_t)head + (phase ? 0 : free) + carry + k;  // below 3 P
        if (i >= a.P) i -= a.P;
        if (i >= a.P) i -= a.P;
        if (phase)
          *cell = a.ring[i];
        else
          a.ring[i] = *cell;
      }
      if (!once) carry += phase ? more.takes : more.gives;
      __syncthreads();
    }
  }

  // lengths and starts last: kv_out may be kv_len
  int64_t carry = 0;
  for (int base = 0; base < a.R; base += THREADS) {
    Request q = mine;
    Sums b = before, more = {};
    if (!once) {
      int f;
      q = request_of(a, base + tid);
      b = scan<THREADS>(q, a.row, more, f, part, flag);
    }
    const int r = base + tid;
    if (r < a.R) {
      const int s = status ? 0 : (int)(carry + b.fresh);
      const int n = status ? a.kv_len[r] : q.kept + q.fresh;
      a.starts[r] = s;
      a.kv_out[r] = n;
      if (once) starts[tid] = s, lens[tid] = n;
    }
    carry += more.fresh;
  }
  if (tid == 0) {
    const int total = status ? 0 : (int)all.fresh;
    a.starts[a.R] = total;
    if (once) starts[a.R] = total;
    int64_t h = status ? head : head + all.takes;
    if (!status && h >= a.P) h -= a.P;
    a.cursor_out[0] = (int)h;
    a.cursor_out[1] = status ? free : (int)(free + all.gives - all.takes);
    a.cursor_out[2] = total;
    a.cursor_out[3] = status;
  }
  if (!once || a.tokens > kSlotsHere) return;
  __syncthreads();
  for (int64_t t = tid; t < a.tokens; t += THREADS)
    map_slot(a, t, [&](int r) { return starts[r]; }, [&](int r) { return lens[r]; });
}

__global__ __launch_bounds__(256) void slot_map_kernel(PlanArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t < a.tokens)
    map_slot(a, t, [&](int r) { return a.starts[r]; }, [&](int r) { return a.kv_out[r]; });
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
  const bool few = R <= kFewRequests;
  const int threads = few ? kFewRequests : kPlanThreads;
  if (few)
    hipLaunchKernelGGL(page_plan_kernel<kFewRequests>, dim3(1), dim3(threads), 0, st, a);
  else
    hipLaunchKernelGGL(page_plan_kernel<kPlanThreads>, dim3(1), dim3(threads), 0, st, a);
  if (int e = launch_status()) return e;
  if (tokens == 0 || (R <= threads && tokens <= kSlotsHere)) return UMIC_OK;
  hipLaunchKernelGGL(slot_map_kernel, dim3((unsigned)((tokens + 255) / 256)), dim3(256), 0, st, a);
  return launch_status();
}
