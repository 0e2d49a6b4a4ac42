// The two operators that fill a paged 8-bit cache: page and slot planning (fa_paged_plan) and the rounding of new keys
// and values into their pages (fa_paged8_append). include/fa_b200.h has the rules that both follow.
#include "fa_paged8.cuh"
#include "fa_sm100.cuh"

#include <atomic>
#include <type_traits>

namespace fa {
namespace {

int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

// ---------------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------------
// Everything follows from three running sums over the requests (new tokens, pages that come back, pages needed): every
// CTA forms them for itself in shared memory, and tokens and pages then find their request there. Where the lengths are
// updated in place the CTAs are one cluster, whose barrier separates the reads of the lengths from the writes. Bound by
// latency (lengths, sums, ids, slots: three trips to memory): 4.4 us for a decode step of 64 requests, 7.9 us for 65613
// tokens of 256 requests (23.5 us with one cluster of eight CTAs and a bisection for every token; updated in place, in one
// cluster, they take 3.2 times as long as in 128 CTAs).
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxCluster = 8;
constexpr int kPlanMaxCtas = 128;

struct PlanArgs {
  int batch, max_blocks, num_blocks, shift, num_tokens;
  const int32_t* lens;
  int64_t cl_stride;
  const int32_t* fresh;
  int64_t nl_stride;
  int32_t* table;
  int64_t bt_stride;
  int32_t* stack;
  const int32_t* count;
  int64_t* slots;
  int32_t* cu;
  int32_t* lens_out;
  int32_t* count_out;
};

enum : uint8_t { kUnserved = 0, kNeedsPages = 1, kEnding = 2, kNoPages = 3 };

__device__ __forceinline__ int saturated(int64_t x) { return (int)min(x, (int64_t)INT32_MAX); }

// Inclusive sums of two values over the CTA; *tx, *ty receive the totals. `part` holds 2 values a warp.
__device__ __forceinline__ void block_scan2(int64_t& x, int64_t& y, int64_t* tx, int64_t* ty, int64_t (*part)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t px = __shfl_up_sync(0xffffffffu, x, o), py = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += px;
      y += py;
    }
  }
  __syncthreads();  // the last call's readers are done with `part`
  if (lane == 31) {
    part[warp][0] = x;
    part[warp][1] = y;
  }
  __syncthreads();
  // every warp adds the warps' totals up for itself (there are at most 32)
  const int warps = blockDim.x >> 5;
  int64_t vx = lane < warps ? part[lane][0] : 0, vy = lane < warps ? part[lane][1] : 0;
  int64_t bx = lane < warp ? vx : 0, by = lane < warp ? vy : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o >= warps) continue;  // (uniform; warps is 1 for a small batch)
    vx += __shfl_xor_sync(0xffffffffu, vx, o);
    vy += __shfl_xor_sync(0xffffffffu, vy, o);
    bx += __shfl_xor_sync(0xffffffffu, bx, o);
    by += __shfl_xor_sync(0xffffffffu, by, o);
  }
  x += __shfl_sync(0xffffffffu, bx, 0);
  y += __shfl_sync(0xffffffffu, by, 0);
  *tx = __shfl_sync(0xffffffffu, vx, 0);
  *ty = __shfl_sync(0xffffffffu, vy, 0);
}

// First index with ends[index] > value (n when there is none), for one value of the whole warp: 32 probes a round.
__device__ __forceinline__ int warp_first_above(const int* ends, int n, int value) {
  const int lane = threadIdx.x & 31;
  int lo = 0, span = n;
  while (span > 0) {
    const int size = (span + 31) >> 5, probe = lo + (lane + 1) * size - 1;  // the last of 32 blocks' elements
    const int below = __popc(__ballot_sync(0xffffffffu, probe < lo + span && ends[probe] <= value));
    lo += below * size;
    span = size == 1 ? 0 : min(size, span - below * size);
  }
  return lo;
}
// The same for a lane's own value, not below the warp's first one, whose index `known` is: within the next 32 entries by
// shuffles, and by bisection in the shared array for lanes that lie behind them (empty entries can be many).
__device__ __forceinline__ int lane_first_above(const int* ends, int n, int known, int value) {
  const int lane = threadIdx.x & 31;
  const int end = known + lane < n ? ends[known + lane] : INT32_MAX;
  int index = 0;
#pragma unroll
  for (int w = 16; w > 0; w >>= 1)
    if (__shfl_sync(0xffffffffu, end, index + w - 1) <= value) index += w;
  if (__shfl_sync(0xffffffffu, end, 31) <= value) {
    int lo = known + 32, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > value) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }
  return known + index;
}

template <int kTogether>
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t part[kPlanThreads / 32][2];
  int* cu_end = reinterpret_cast<int*>(smem);
  int* need_end = cu_end + a.batch;
  int* back_end = need_end + a.batch;
  int* len = back_end + a.batch;
  uint8_t* state = reinterpret_cast<uint8_t*>(len + a.batch);
  const int tid = threadIdx.x, threads = blockDim.x;
  grid_launch_dependents();
  grid_dependency_wait();  // (launched while the kernel before it ends)
  const int64_t round_up = (1 << a.shift) - 1, capacity = (int64_t)a.max_blocks << a.shift;
  const int count = max(0, min(*a.count, a.num_blocks));

  int64_t fresh_sum = 0, back_sum = 0, need_sum = 0;
  for (int c = 0; c < a.batch; c += threads) {
    const int b = c + tid;
    const bool in = b < a.batch;
    const int64_t L = in ? a.lens[b * a.cl_stride] : 0, n = in ? a.fresh[b * a.nl_stride] : 0;
    int64_t fresh = max(n, (int64_t)0), tf, tb;
    int64_t back = n < 0 && L > 0 ? min((L + round_up) >> a.shift, (int64_t)a.max_blocks) : 0;
    block_scan2(fresh, back, &tf, &tb, part);
    const bool fits = in && n >= 0 && L >= 0 && L + n <= capacity && fresh_sum + fresh <= a.num_tokens;
    const int64_t mine = fits ? ((L + n + round_up) >> a.shift) - ((L + round_up) >> a.shift) : 0;
    int64_t need = mine, unused = 0, tn, tu;
    block_scan2(need, unused, &tn, &tu, part);
    if (in) {
      cu_end[b] = saturated(fresh_sum + fresh);
      back_end[b] = saturated(back_sum + back);
      need_end[b] = saturated(need_sum + need);
      len[b] = (int)L;
      state[b] = n < 0 ? kEnding : !fits ? kUnserved : mine > 0 ? kNeedsPages : kNoPages;
    }
    fresh_sum += tf;
    back_sum += tb;
    need_sum += tn;
  }
  // (below the value that running sums stop at, so that a request behind 2^31 needed pages is never taken for served)
  const int available = (int)min(count + back_sum, (int64_t)INT32_MAX - 1);
  __syncthreads();
  for (int b = tid; b < a.batch; b += threads)
    if (state[b] == kNeedsPages && need_end[b] > available) state[b] = kUnserved;
  __syncthreads();
  // every CTA has read the lengths and the count (and finished its own sums) before anyone writes
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");

  const int first = blockIdx.x * threads + tid, step = gridDim.x * threads;
  const int lane = tid & 31;
  // pages taken: the running need of the last request that is within what the stack holds
  const int served_below = warp_first_above(need_end, a.batch, available);
  const int taken = served_below > 0 ? need_end[served_below - 1] : 0;
  const int left = available - taken;

  // Place `from` of the stack once the pages of ending requests lie on top of it. Nothing that is read here is written by
  // this call: the stack below its old top, pages that requests held before, rows of ending requests.
  auto entry = [&](int from) -> const int32_t* {
    if (from < count) return a.stack + from;
    const int k = from - count;
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (back_end[mid] > k) hi = mid;
      else lo = mid + 1;
    }
    return a.table + (int64_t)lo * a.bt_stride + (k - (lo > 0 ? back_end[lo - 1] : 0));
  };

  // Slots, in groups of 32 tokens, kTogether of them at a time so that the loads of their page ids overlap. A group that
  // lies in the request of the token before it needs no search; otherwise every lane looks for its own.
  for (int64_t t0 = (int64_t)(first - lane) * kTogether; t0 < a.num_tokens; t0 += (int64_t)step * kTogether) {
    const int32_t* from[kTogether];
    int id[kTogether], offset[kTogether], known = warp_first_above(cu_end, a.batch, (int)t0);
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int64_t t_last = t0 + 32 * k + 31;
      from[k] = nullptr;
      offset[k] = 0;
      if (t0 + 32 * k >= a.num_tokens) continue;
      const int t = (int)min(t0 + 32 * k + lane, (int64_t)a.num_tokens - 1);
      int b = known;
      if (known < a.batch && cu_end[known] <= t_last) {
        b = lane_first_above(cu_end, a.batch, known, t);
        known = __shfl_sync(0xffffffffu, b, 31);
      }
      if (b >= a.batch || (state[b] != kNeedsPages && state[b] != kNoPages)) continue;
      const int pos = len[b] + (t - (b > 0 ? cu_end[b - 1] : 0));
      const int page = pos >> a.shift, have = (int)((len[b] + round_up) >> a.shift);
      offset[k] = pos & (int)round_up;
      from[k] = page < have ? a.table + (int64_t)b * a.bt_stride + page
                            : entry(available - 1 - (b > 0 ? need_end[b - 1] : 0) - (page - have));
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) id[k] = from[k] != nullptr ? *from[k] : -1;
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
      if (t0 + 32 * k + lane < a.num_tokens)
        a.slots[t0 + 32 * k + lane] = id[k] >= 0 && id[k] < a.num_blocks ? ((int64_t)id[k] << a.shift) + offset[k] : -1;
  }
  // block-table entries of the new pages, and the places of the stack above its old top
  // (counted in 64 bits: a stack may hold up to 2^31 - 1 pages, and the last step leads past that)
  for (int64_t p0 = first - lane; p0 < taken; p0 += step) {
    const int p = (int)min(p0 + lane, (int64_t)taken - 1);
    const int b = lane_first_above(need_end, a.batch, warp_first_above(need_end, a.batch, (int)p0), p);
    const int have = (int)((len[b] + round_up) >> a.shift);
    if (p0 + lane < taken)
      a.table[(int64_t)b * a.bt_stride + have + (p - (b > 0 ? need_end[b - 1] : 0))] = *entry(available - 1 - p);
  }
  for (int64_t p = (int64_t)count + first; p < min(left, a.num_blocks); p += step) a.stack[p] = *entry((int)p);
  for (int b = first; b < a.batch; b += step) {
    const int begin = b > 0 ? cu_end[b - 1] : 0;
    a.cu[b + 1] = cu_end[b];
    a.lens_out[b] = state[b] == kEnding ? 0 : state[b] == kUnserved ? len[b] : len[b] + (cu_end[b] - begin);
  }
  if (first == 0) {
    a.cu[0] = 0;
    *a.count_out = min(left, a.num_blocks);
  }
}

// ---------------------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------------------
// A task is the run of new tokens of one page, for one head, of keys or of values. Its rows stay in registers between
// the maximum and the rounding (up to 8 loads of 16 bytes a lane and `warps` warps a task; longer runs are read twice).
// A CTA holds 8 / warps tasks of the same runs: the heads of a token are neighbours in memory. Bound by memory with many
// tokens, but only where few instructions go to a value: 45.5 us for 32704 tokens of 16 heads of 64, fp16 -> int8 (201 MB,
// 4.4 TB/s, 67 % of a plain copy's rate), 14 us for 8192 tokens of 8 heads of 128, bf16 -> e4m3 (50 MB, 3.6 TB/s); 13
// instructions a value before the folded maxima and the 16-bit arithmetic: 64 and 18 us. A decode step of 128 requests
// takes 4 us. 80 registers hold the rows and leave 24 warps an SM; reading them again instead (64 or 40 registers) takes
// 59 and 78 us.
constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kAppendLoads = 8;
constexpr int kAppendWindow = 512;  // slots that a CTA looks at: up to 256 that may start a run, and those behind them

struct AppendArgs {
  int heads, head_dim, shift, range, warps;  // range: tokens whose runs a CTA starts; warps: warps a task
  int64_t num_tokens, num_slots;
  const void* src[2];
  int64_t src_st[2], src_sh[2];
  uint8_t* cache[2];
  int64_t c_sb[2], c_st[2], c_sh[2];
  float* scales[2];
  int64_t s_sb[2], s_sh[2];
  const int64_t* slots;
  int64_t slot_stride;
  int32_t* status;
};

template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };

// Eight 16-bit values as four pairs' magnitudes, into the running largest of each pair (NaN wins).
template <typename T>
__device__ __forceinline__ void amax8(const uint4& v, typename Pair<T>::type (&m)[4]) {
  using P = typename Pair<T>::type;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = __hmax2_nan(m[i], __habs2(*reinterpret_cast<const P*>(&w[i])));
}
// Largest finite magnitude of eight 16-bit values, some of which are not.
template <typename T>
__device__ __noinline__ float finite_amax8(const uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float best = 0.f;
  for (int i = 0; i < 4; ++i) {
    const float2 f = DType<T>::unpack2(w[i]);
    if (fabsf(f.x) < INFINITY) best = fmaxf(best, fabsf(f.x));
    if (fabsf(f.y) < INFINITY) best = fmaxf(best, fabsf(f.y));
  }
  return best;
}

// Smallest power of two s >= 2^-126 with amax <= s * largest code.
template <typename C8>
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - C8::kTopExp + ((u & 0x7fffffu) > C8::kTopMant ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Four 16-bit values -> four codes: times the inverse of a power of two (finite values; kHalf: fp16 values, and an inverse
// that is an fp16 number, in fp16 arithmetic that rounds once), or divided by any scale.
template <typename T, typename C8, bool kHalf>
__device__ __forceinline__ uint32_t scaled4(uint32_t lo, uint32_t hi, float inverse) {
  if constexpr (kHalf) {
    const __half2 f = __float2half2_rn(inverse);
    return C8::pack4_half(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&hi), f);
  }
  const float2 x = DType<T>::unpack2(lo), y = DType<T>::unpack2(hi);
  return C8::pack4_times(x.x, x.y, y.x, y.y, inverse);
}
__device__ __forceinline__ float divided(float x, float scale) {
  if (scale < 0x1p-60f) {  // (the rest of a division by a tiny scale would be below fp32's range)
    x *= 0x1p60f;
    scale *= 0x1p60f;
  }
  const float q = __fdiv_rz(x, scale);
  return to_odd(q, fmaf(-q, scale, x));
}
template <typename T, typename C8>
__device__ __noinline__ uint32_t divided4(uint32_t lo, uint32_t hi, float scale) {
  const float2 x = DType<T>::unpack2(lo), y = DType<T>::unpack2(hi);
  return C8::pack4(divided(x.x, scale), divided(x.y, scale), divided(y.x, scale), divided(y.y, scale));
}

template <typename T, typename C8, bool kWide>
__global__ void __launch_bounds__(kAppendThreads, 3) paged8_append_kernel(const AppendArgs a) {
  __shared__ float part[2][kAppendWarps];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int bs = 1 << a.shift;
  __shared__ int64_t slot_s[kWide ? kAppendWindow + 1 : 1];  // from the token in front of the range on; -1: none
  __shared__ int16_t start_s[kAppendThreads];
  __shared__ int count_s[kAppendWarps];
  [[maybe_unused]] const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.range;
  const int task = blockIdx.y * (kAppendWarps / a.warps) + warp / a.warps, turn = warp % a.warps;
  const bool has_task = task < 2 * a.heads;
  const int kv = has_task ? task / a.heads : 0, head = has_task ? task % a.heads : 0;
  const int lanes = a.head_dim / 8, rows = 32 / lanes;  // lanes a row of 16-bit values, rows a load
  const int row = lane / lanes, col = lane % lanes;
  const char* src = reinterpret_cast<const char*>(a.src[kv]) + (head * a.src_sh[kv] + col * 8) * 2;
  uint8_t* cache = a.cache[kv] + head * a.c_sh[kv];
  const int lanes8 = a.head_dim / 16, rows8 = 32 / lanes8;

  // Runs that start in [t0, t0 + range): neighbours with slots in the same page.
  auto slot_at = [&](int64_t t) -> int64_t {
    const int64_t s = t >= 0 && t < a.num_tokens ? a.slots[t * a.slot_stride] : -1;
    return s >= 0 && s < a.num_slots ? s : -1;
  };
  // A warp a task (kWide false): every warp finds the runs by itself, and none waits for another. Several warps a task, pages
  // of more tokens: the CTA finds them together, over ranges of up to 256 tokens.
  int64_t s = -1;
  uint32_t starts = 0u, breaks = 0u;
  bool disorder = false;
  int runs = 0;
  const int window = min(a.range + bs, kAppendWindow);
  if constexpr (!kWide) {
    s = slot_at(t0 + lane);
    int64_t before = __shfl_up_sync(0xffffffffu, s, 1);
    if (lane == 0) before = slot_at(t0 - 1);
    const bool same = s >= 0 && before >= 0 && (s >> a.shift) == (before >> a.shift);
    disorder = same && s != before + 1;
    starts = __ballot_sync(0xffffffffu, s >= 0 && !same && lane < a.range);
    breaks = __ballot_sync(0xffffffffu, !same);
    runs = __popc(starts);
  } else {
    for (int i = tid; i <= window; i += kAppendThreads) slot_s[i] = slot_at(t0 - 1 + i);
    __syncthreads();
    {
      const int64_t mine = tid < a.range ? slot_s[tid + 1] : -1, before = slot_s[min(tid, window)];
      const bool same = mine >= 0 && before >= 0 && (mine >> a.shift) == (before >> a.shift);
      disorder = same && mine != before + 1;
      const bool start = mine >= 0 && !same;
      const uint32_t mask = __ballot_sync(0xffffffffu, start);
      if (lane == 0) count_s[warp] = __popc(mask);
      __syncthreads();
      int at = __popc(mask & ((1u << lane) - 1));
      for (int w = 0; w < warp; ++w) at += count_s[w];
      if (start) start_s[at] = (int16_t)tid;
    }
    __syncthreads();
    for (int w = 0; w < kAppendWarps; ++w) runs += count_s[w];
  }
  if (disorder && a.status != nullptr) *a.status = FA_STATUS_SLOT_ORDER;

  int parity = 0;
  // Runs that a warp holds alone (a decode step's single tokens) are dealt to the task's warps, then all of them share each
  // longer one.
  for (int pass = 0; pass < (kWide ? 2 : 1); ++pass)
  for (int run = kWide && pass == 0 ? turn : 0; run < runs; run += kWide && pass == 0 ? a.warps : 1) {
    const int warps = kWide && pass == 1 ? a.warps : 1, sub = kWide && pass == 1 ? turn : 0;
    const int chunk = kAppendLoads * rows * warps;  // tokens that these warps hold at once
    int i;
    int64_t slot;
    if constexpr (!kWide) {
      i = __ffs(starts) - 1;
      starts &= starts - 1;
      slot = __shfl_sync(0xffffffffu, s, i);
    } else {
      i = start_s[run];
      slot = slot_s[i + 1];
    }
    const int64_t page = slot >> a.shift, t_first = t0 + i;
    const int offset = (int)(slot & (bs - 1));
    int n;
    if constexpr (!kWide) {
      const uint32_t later = i == 31 ? 0u : breaks & (0xffffffffu << (i + 1));
      if (later) {
        n = __ffs(later) - 1 - i;
      } else {
        n = 32 - i;
        for (int64_t t = t0 + 32; n < bs; t += 32) {  // the run leaves the window
          const int64_t x = slot_at(t + lane);
          const bool cont = x >= 0 && (x >> a.shift) == page;
          const uint32_t stop = __ballot_sync(0xffffffffu, !cont);
          const int more = stop ? __ffs(stop) - 1 : 32;
          n += more;
          if (stop) break;
        }
      }
    } else {
      n = 1;
      for (; n < bs - offset; n += 32) {
        const int x = i + n + lane;
        const int64_t next = x < window ? slot_s[x + 1] : slot_at(t0 + x);
        const uint32_t stop = __ballot_sync(0xffffffffu, next < 0 || (next >> a.shift) != page);
        if (stop) {
          n += __ffs(stop) - 1;
          break;
        }
      }
    }
    n = min(n, bs - offset);
    if (kWide && (n > kAppendLoads * rows) != (pass == 1)) continue;

    // ---- largest magnitude of the run
    using P = typename Pair<T>::type;
    const int64_t row_bytes = a.src_st[kv] * 2, load_step = rows * row_bytes;
    const char* mine = src + t_first * row_bytes + (sub * kAppendLoads * rows + row) * row_bytes;
    const int first_j = sub * kAppendLoads * rows + row, end_j = has_task && row < rows ? n : 0;  // a lane's rows, up to end_j
    uint4 held[kAppendLoads];
    const uint32_t none = 0u;
    P m[4] = {*reinterpret_cast<const P*>(&none), *reinterpret_cast<const P*>(&none), *reinterpret_cast<const P*>(&none),
              *reinterpret_cast<const P*>(&none)};
    for (int base = 0; base < n; base += chunk) {
      const char* at = mine + base * row_bytes;
#pragma unroll
      for (int l = 0; l < kAppendLoads; ++l, at += load_step) {
        held[l] = make_uint4(0u, 0u, 0u, 0u);
        if (first_j + base + l * rows < end_j) held[l] = __ldg(reinterpret_cast<const uint4*>(at));
      }
#pragma unroll
      for (int l = 0; l < kAppendLoads; ++l) amax8<T>(held[l], m);
    }
    const P both = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
    float amax = fmaxf(DType<T>::to_float(both.x), DType<T>::to_float(both.y));
    const bool special = !(DType<T>::to_float(both.x) < INFINITY && DType<T>::to_float(both.y) < INFINITY);
    if (special) {  // again, over the finite ones alone
      amax = 0.f;
      for (int j = first_j; j < end_j; j += rows) {
        const int l = (j - first_j) / rows;
        if (l % (kAppendLoads * warps) >= kAppendLoads) continue;  // other warps' rows
        amax = fmaxf(amax, finite_amax8<T>(__ldg(reinterpret_cast<const uint4*>(mine + l * load_step))));
      }
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    float* scale_at = a.scales[kv] + page * a.s_sb[kv] + head * a.s_sh[kv];
    const float old = offset > 0 ? *scale_at : 0.f;
    if (kWide && pass == 1) {
      if (lane == 0) part[parity][warp] = amax;
      __syncthreads();  // also: every warp of the task has read the old scale
      for (int w = 0; w < warps; ++w) amax = fmaxf(amax, part[parity][warp - sub + w]);
      parity ^= 1;
    }
    __syncwarp();
    const float wanted = scale_for<C8>(amax);
    const float scale = offset > 0 ? fmaxf(old, wanted) : wanted;
    if (!has_task) continue;
    if (sub == 0 && lane == 0) *scale_at = scale;
    uint8_t* page_base = cache + page * a.c_sb[kv];

    // ---- older tokens of the page, when its scale has grown
    if (offset > 0 && scale != old) {
      const float ratio = __fdiv_rn(old, scale);  // (exact: the scale has grown to a power of two)
      const int r8 = lane / lanes8, c8 = lane % lanes8;
      for (int j = sub * rows8 + r8; r8 < rows8 && j < offset; j += warps * rows8) {
        uint4* at = reinterpret_cast<uint4*>(page_base + j * a.c_st[kv] + c8 * 16);
        uint4 v = *at;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 lo = DType<__half>::unpack2(C8::lo(w[k])), hi = DType<__half>::unpack2(C8::hi(w[k]));
          w[k] = C8::pack4_codes(lo, hi, ratio);
        }
        *at = v;
      }
    }

    // ---- the new tokens. Dividing by a power of two is multiplying by its inverse; a scale that the caller made and
    // that is none is divided by.
    const bool simple = (__float_as_uint(scale) & 0x7fffffu) == 0 && !__any_sync(0xffffffffu, special);
    const float inverse = __fdiv_rn(1.f, scale);
    const int64_t store_step = rows * a.c_st[kv];
    for (int base = 0; base < n; base += chunk) {
      const char* at = mine + base * row_bytes;
      uint8_t* to = page_base + (int64_t)(offset + base + first_j) * a.c_st[kv] + col * 8;
      if (simple) {
        if (n > chunk) {
          const char* again = at;
#pragma unroll
          for (int l = 0; l < kAppendLoads; ++l, again += load_step)
            if (first_j + base + l * rows < end_j) held[l] = __ldg(reinterpret_cast<const uint4*>(again));
        }
        auto store = [&](auto half) {
#pragma unroll
          for (int l = 0; l < kAppendLoads; ++l, to += store_step)
            if (first_j + base + l * rows < end_j)
              *reinterpret_cast<uint2*>(to) = make_uint2(scaled4<T, C8, decltype(half)::value>(held[l].x, held[l].y, inverse),
                                                         scaled4<T, C8, decltype(half)::value>(held[l].z, held[l].w, inverse));
        };
        if (std::is_same<T, __half>::value && inverse <= 32768.f && inverse >= 6.103515625e-05f)
          store(std::integral_constant<bool, std::is_same<T, __half>::value>());
        else
          store(std::false_type());
      } else {
#pragma unroll 1
        for (int l = 0; l < kAppendLoads; ++l, to += store_step)
          if (first_j + base + l * rows < end_j) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(at + l * load_step));
            *reinterpret_cast<uint2*>(to) = make_uint2(divided4<T, C8>(v.x, v.y, scale), divided4<T, C8>(v.z, v.w, scale));
          }
      }
    }
  }
}

int check_launch(const char* what, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  return e == cudaSuccess ? 0 : set_error(FA_ERR_LAUNCH, "%s launch failed: %s", what, cudaGetErrorString(e));
}

// The shared memory of the largest batch, allowed once a device and never lowered: calls of other threads may be on their
// way to a launch.
constexpr int kPlanBytes = 17;  // shared memory of a request
constexpr int kMaxDevices = 64;
template <int kTogether> int allow_plan_smem() {
  static std::atomic<bool> allowed[kMaxDevices];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < kMaxDevices && allowed[dev].load(std::memory_order_relaxed)) return 0;
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(paged_plan_kernel<kTogether>, cudaFuncAttributeMaxDynamicSharedMemorySize, FA_PLAN_MAX_BATCH * kPlanBytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(FA_ERR_LAUNCH, "plan: cannot get %d bytes of shared memory: %s", FA_PLAN_MAX_BATCH * kPlanBytes, cudaGetErrorString(e));
  }
  if (dev < kMaxDevices) allowed[dev].store(true, std::memory_order_relaxed);
  return 0;
}

}  // namespace

int launch_paged_plan(const fa_paged_plan_params& p, cudaStream_t stream) {
  if (p.num_tokens > INT32_MAX || ((int64_t)p.max_blocks * p.block_size) > INT32_MAX)
    return set_error(FA_ERR_UNSUPPORTED, "plan: more than 2^31 - 1 tokens");
  PlanArgs a = {};
  a.batch = p.batch;
  a.max_blocks = p.max_blocks;
  a.num_blocks = p.num_blocks;
  a.shift = log2_of(p.block_size);
  a.num_tokens = (int)p.num_tokens;
  a.lens = p.context_lens;
  a.cl_stride = p.cl_stride;
  a.fresh = p.new_lens;
  a.nl_stride = p.nl_stride;
  a.table = p.block_table;
  a.bt_stride = p.bt_stride;
  a.stack = p.free_blocks;
  a.count = p.free_count;
  a.slots = p.slot_mapping;
  a.cu = p.cu_seqlens;
  a.lens_out = p.context_lens_out;
  a.count_out = p.free_count_out;
  const bool inplace = a.lens_out == a.lens || a.count_out == a.count;
  const int smem = p.batch * kPlanBytes;
  if (smem > 40 * 1024) {
    const int rc = inplace ? allow_plan_smem<4>() : allow_plan_smem<1>();
    if (rc) return rc;
  }
  // A thread for each request or token of a decode step; more CTAs for prompts, as many as there are groups of tokens for
  // where the lengths are not updated in place, a cluster that takes four groups at a time where they are.
  const int64_t work = p.num_tokens > p.batch ? p.num_tokens : p.batch;
  const int threads = work >= kPlanThreads ? kPlanThreads : (int)((work + 31) / 32 * 32);
  int ctas = 1;
  while (ctas < (inplace ? kPlanMaxCluster : kPlanMaxCtas) && ctas * kPlanThreads < work) ctas *= 2;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = ctas;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attrs;
  cfg.numAttrs = inplace ? 2 : 1;
  return check_launch("plan", inplace ? cudaLaunchKernelEx(&cfg, paged_plan_kernel<4>, a)
                                      : cudaLaunchKernelEx(&cfg, paged_plan_kernel<1>, a));
}

int launch_paged8_append(const fa_paged8_append_params& p, cudaStream_t stream) {
  AppendArgs a = {};
  a.heads = p.heads_kv;
  a.head_dim = p.head_dim;
  a.shift = log2_of(p.block_size);
  a.num_tokens = p.num_tokens;
  a.num_slots = (int64_t)p.num_blocks * p.block_size;
  a.src[0] = p.key;
  a.src[1] = p.value;
  a.src_st[0] = p.key_strides[0];
  a.src_sh[0] = p.key_strides[1];
  a.src_st[1] = p.value_strides[0];
  a.src_sh[1] = p.value_strides[1];
  a.cache[0] = static_cast<uint8_t*>(p.k_cache);
  a.cache[1] = static_cast<uint8_t*>(p.v_cache);
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t* st = kv ? p.v_strides : p.k_strides;
    const int64_t* ss = kv ? p.vs_strides : p.ks_strides;
    a.c_sb[kv] = st[0];
    a.c_st[kv] = st[1];
    a.c_sh[kv] = st[2];
    a.scales[kv] = kv ? p.v_scales : p.k_scales;
    a.s_sb[kv] = ss[0];
    a.s_sh[kv] = ss[1];
  }
  a.slots = p.slot_mapping;
  a.slot_stride = p.slot_stride;
  a.status = p.status;
  const int rows = 32 / (p.head_dim / 8);
  a.warps = 1;
  while (a.warps < kAppendWarps && a.warps * kAppendLoads * rows < p.block_size) a.warps *= 2;
  // (a few tokens are the single ones of a decode step: no more warps a task than there is room for at once)
  while (a.warps > 1 && p.num_tokens <= 256 && p.num_tokens * 2 * p.heads_kv * a.warps > 148 * 3 * kAppendWarps) a.warps /= 2;
  const int64_t tasks = (2 * p.heads_kv + kAppendWarps / a.warps - 1) / (kAppendWarps / a.warps);
  if (tasks > 65535) return set_error(FA_ERR_UNSUPPORTED, "append: too many heads");
  // a CTA starts the runs of `range` tokens: one while the grid is small, up to a page's (at most 256) for prompts
  a.range = 1;
  const bool wide = a.warps > 1;
  while (a.range < (wide ? kAppendThreads : 32) && a.range < p.block_size && p.num_tokens * tasks / (2 * a.range) >= 592) a.range *= 2;
  const int64_t grid = (p.num_tokens + a.range - 1) / a.range;
  if (grid > INT32_MAX) return set_error(FA_ERR_UNSUPPORTED, "append: too many tokens");
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, (unsigned)tasks);
  cfg.blockDim = dim3(kAppendThreads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const bool e4m3 = p.cache_dtype == FA_CACHE_E4M3, fp16 = p.dtype == FA_F16;
  cudaError_t e;
  if (wide) {
    if (fp16) e = e4m3 ? cudaLaunchKernelEx(&cfg, paged8_append_kernel<__half, CodeE4M3, true>, a)
                       : cudaLaunchKernelEx(&cfg, paged8_append_kernel<__half, CodeInt8, true>, a);
    else e = e4m3 ? cudaLaunchKernelEx(&cfg, paged8_append_kernel<__nv_bfloat16, CodeE4M3, true>, a)
                  : cudaLaunchKernelEx(&cfg, paged8_append_kernel<__nv_bfloat16, CodeInt8, true>, a);
  } else {
    if (fp16) e = e4m3 ? cudaLaunchKernelEx(&cfg, paged8_append_kernel<__half, CodeE4M3, false>, a)
                       : cudaLaunchKernelEx(&cfg, paged8_append_kernel<__half, CodeInt8, false>, a);
    else e = e4m3 ? cudaLaunchKernelEx(&cfg, paged8_append_kernel<__nv_bfloat16, CodeE4M3, false>, a)
                  : cudaLaunchKernelEx(&cfg, paged8_append_kernel<__nv_bfloat16, CodeInt8, false>, a);
  }
  return check_launch("append", e);
}

}  // namespace fa
