// Page tables, token slots and positions of a serving step, from the requests' lengths.
//
// Request r holds cached[r] tokens in its first ceil(cached / page) table entries and appends
// new[r] tokens (new[r] = -1: it is finished and gives its pages back).  Pages come from and go
// to a ring of free pages; ring[0] / ring[1] count the pages ever taken from / put into it, so
// the free ones are entries ring[0] .. ring[1] - 1 modulo its size.  With need_r new pages of
// request r and U_r = sum_{q <= r} need_q, request r is served when U_r pages are free: its
// pages are entries ring[0] + U_r - need_r ..; a request that is not served keeps its length and
// its tokens get no slot.  Finished requests' pages are appended behind ring[1], in order.
//
// The work is three prefix sums over the requests (tokens, pages taken, pages returned) and one
// short computation per token and per moved page.  Every CTA runs the prefix sums over all
// requests, 1024 at a time, and takes every gridDim-th group of 1024 tokens and pages, which it
// finds by bisection in the prefix sums of the chunk: no second launch and no wait between CTAs.
//
// Bound by latency, a chain of dependent loads and barriers per chunk: 256 decoding requests 7.3 us;
// 1500 requests with 16381 tokens of prompts, two chunks, 23 us (0.5 MB).
#include "params.cuh"

namespace dsv2 {

constexpr int kPlanThreads = 1024;

struct PlanScan {
  long long tok, need, back;
};

__device__ __forceinline__ PlanScan plan_shfl_up(const PlanScan& v, int o) {
  return {__shfl_up_sync(0xffffffffu, v.tok, o), __shfl_up_sync(0xffffffffu, v.need, o),
          __shfl_up_sync(0xffffffffu, v.back, o)};
}

// largest i in [0, n) with s[i] <= v (s ascending, s[0] <= v)
__device__ __forceinline__ int plan_find(const long long* s, int n, long long v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(const PagePlanParams p) {
  pdl_enter();
  __shared__ long long s_tok[kPlanThreads + 1], s_need[kPlanThreads + 1], s_back[kPlanThreads + 1];
  __shared__ PlanScan s_warp[32];
  __shared__ int s_cached[kPlanThreads], s_flags[kPlanThreads];   // flags: 1 served, 2 finished
  __shared__ int s_ticket, s_deferred;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long grid = gridDim.x, cta = blockIdx.x;
  const long long head = p.ring_in[0], tail = p.ring_in[1];
  const bool ring_ok = tail >= head && tail - head <= p.ring_size && head >= 0;
  const long long avail = ring_ok ? tail - head : 0;
  if (tid == 0) s_deferred = 0;
  if (cta == 0 && tid == 0) p.cu_new[0] = 0;
  __syncthreads();   // every thread has read ring_in
  if (tid == 0) {
    // the CTA that read the counters last writes the new ones: ring_out may be ring_in
    __threadfence();
    s_ticket = atomicAdd(p.sync, 1);
    if (!ring_ok) set_device_error(kErrIndex);
  }
  PlanScan base = {0, 0, 0};
  long long taken = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kPlanThreads) {
    const int n = min(kPlanThreads, p.requests - r0), r = r0 + tid;
    // --- this chunk's requests
    PlanScan v = {0, 0, 0};
    int cached = 0, fresh = 0, kept = 0;   // kept: the length that a request which is not served keeps
    bool finished = false, fits = false;
    if (tid < n) {
      const long long c = p.cached64 ? reinterpret_cast<const long long*>(p.cached)[r] : reinterpret_cast<const int*>(p.cached)[r];
      const int nw = p.fresh[r];
      const long long most = static_cast<long long>(p.width) * p.page;
      const bool ok = c >= 0 && c <= most && nw >= -1;
      finished = ok && nw < 0;
      cached = ok ? static_cast<int>(c) : 0;
      kept = static_cast<int>(min(max(c, -0x80000000LL), 0x7fffffffLL));
      fresh = ok ? max(nw, 0) : 0;
      fits = ok && nw >= 0 && c + fresh <= most;
      if (!ok || (nw >= 0 && !fits)) set_device_error(kErrIndex);
      const long long held = (cached + static_cast<long long>(p.page) - 1) / p.page;
      v.tok = fresh;
      v.need = fits ? (cached + static_cast<long long>(fresh) + p.page - 1) / p.page - held : 0;
      v.back = finished ? held : 0;
    }
    const PlanScan mine = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const PlanScan u = plan_shfl_up(v, o);
      if (lane >= o) {
        v.tok += u.tok;
        v.need += u.need;
        v.back += u.back;
      }
    }
    __syncthreads();   // the previous chunk is done with the shared arrays
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      PlanScan w = s_warp[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const PlanScan u = plan_shfl_up(w, o);
        if (lane >= o) {
          w.tok += u.tok;
          w.need += u.need;
          w.back += u.back;
        }
      }
      s_warp[lane] = w;
    }
    __syncthreads();
    if (warp > 0) {
      v.tok += s_warp[warp - 1].tok;
      v.need += s_warp[warp - 1].need;
      v.back += s_warp[warp - 1].back;
    }
    const PlanScan total = s_warp[31];
    s_tok[tid] = base.tok + v.tok - mine.tok;      // exclusive
    s_need[tid] = base.need + v.need - mine.need;
    s_back[tid] = base.back + v.back - mine.back;
    const bool served = fits && base.tok + v.tok <= p.capacity && (mine.need == 0 || base.need + v.need <= avail);
    s_cached[tid] = cached;
    s_flags[tid] = (served ? 1 : 0) | (finished ? 2 : 0);
    if (tid == 0) {
      s_tok[n] = base.tok + total.tok;
      s_need[n] = base.need + total.need;
      s_back[n] = base.back + total.back;
    }
    const long long upto = served && mine.need > 0 ? base.need + v.need : 0;
    if (tid < n && !served && !finished) atomicAdd(&s_deferred, 1);
    if (cta == (r0 / kPlanThreads) % grid && tid < n) {
      p.lens[r] = finished ? 0 : (served ? cached + fresh : kept);
      p.cu_new[r + 1] = static_cast<int>(min(base.tok + v.tok, 0x7fffffffLL));
    }
    // pages taken: the largest U_r of a served request (served requests that need pages come first)
    long long best = upto;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();   // the prefix sums are complete; s_warp is free again
    if (lane == 0) s_warp[warp].tok = best;
    // --- tokens of the chunk, in groups of kPlanThreads
    const long long t_end = min(s_tok[n], static_cast<long long>(p.capacity));
    for (long long g = base.tok / kPlanThreads; g * kPlanThreads < t_end; ++g) {
      if (g % grid != cta) continue;
      const long long t = g * kPlanThreads + tid;
      if (t < base.tok || t >= t_end) continue;
      const int i = plan_find(s_tok, n, t);
      const long long pos = s_cached[i] + (t - s_tok[i]);
      const bool ok = (s_flags[i] & 1) != 0;
      long long slot = -1;
      if (ok) {
        const long long k = pos / p.page, held = (s_cached[i] + static_cast<long long>(p.page) - 1) / p.page;
        const long long pg = k < held ? p.table[static_cast<long long>(r0 + i) * p.table_stride + k]
                                      : p.ring[(head + s_need[i] + (k - held)) % p.ring_size];
        slot = pg * p.page + pos % p.page;
      }
      p.token_row[t] = r0 + i;
      p.positions[t] = ok ? pos : -1;
      p.slots[t] = slot;
    }
    // --- pages the chunk takes
    const long long n_end = min(s_need[n], avail);
    for (long long g = base.need / kPlanThreads; g * kPlanThreads < n_end; ++g) {
      if (g % grid != cta) continue;
      const long long u = g * kPlanThreads + tid;
      if (u < base.need || u >= n_end) continue;
      const int i = plan_find(s_need, n, u);
      if (!(s_flags[i] & 1)) continue;
      const long long held = (s_cached[i] + static_cast<long long>(p.page) - 1) / p.page;
      p.table[static_cast<long long>(r0 + i) * p.table_stride + held + (u - s_need[i])] = p.ring[(head + u) % p.ring_size];
    }
    // --- pages the chunk returns
    for (long long g = base.back / kPlanThreads; g * kPlanThreads < s_back[n]; ++g) {
      if (g % grid != cta) continue;
      const long long u = g * kPlanThreads + tid;
      if (u < base.back || u >= s_back[n]) continue;
      const int i = plan_find(s_back, n, u);
      if (!ring_ok || avail + u >= p.ring_size) {   // more pages than the ring ever held
        set_device_error(kErrIndex);
        continue;
      }
      p.ring[(tail + u) % p.ring_size] = p.table[static_cast<long long>(r0 + i) * p.table_stride + (u - s_back[i])];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 32; ++w) taken = max(taken, s_warp[w].tok);
    base.tok += total.tok;
    base.need += total.need;
    base.back += total.back;
  }
  // --- token rows past the last token
  for (long long t = cta * kPlanThreads + tid; t < p.capacity; t += grid * kPlanThreads) {
    if (t < base.tok) continue;
    p.token_row[t] = -1;
    p.positions[t] = -1;
    p.slots[t] = -1;
  }
  if (tid == 0 && s_ticket == grid - 1) {
    *p.sync = 0;
    const long long back = ring_ok ? min(base.back, p.ring_size - avail) : 0;
    p.ring_out[0] = head + taken;
    p.ring_out[1] = tail + back;
    p.counts[0] = static_cast<int>(min(base.tok, 0x7fffffffLL));
    p.counts[1] = static_cast<int>(taken);
    p.counts[2] = static_cast<int>(back);
    p.counts[3] = s_deferred;
  }
}

cudaError_t launch_page_plan(const PagePlanParams& p, int num_sms, cudaStream_t st) {
  const long long most = std::max<long long>(p.capacity, p.requests);
  const long long groups = (most + kPlanThreads - 1) / kPlanThreads;
  const int grid = static_cast<int>(std::min<long long>(std::max<long long>(groups, 1), num_sms));
  launch_kernel(page_plan_kernel, grid, kPlanThreads, 0, st, p);
  return cudaGetLastError();
}

}  // namespace dsv2
