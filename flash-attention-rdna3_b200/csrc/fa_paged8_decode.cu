// Decode attention over a paged 8-bit cache (fa_decode_paged8).
//
//   o = sum_t p_t vs_t v_t / sum_t p_t,   p_t = 2^(s_t - m),   s_t = log2(e) * softmax_scale * ks_t * (q . k_t)
//
// with ks_t, vs_t the scales of the page that holds token t. One pass over the cache with running m and sums; every byte
// is read once for all query heads of its kv head, so the bound is HBM: 2 * head_dim bytes a token and kv head.
//
// One CTA an SM: a producer warp brings tiles of 64 KB (64, 32 or 16 tokens of 8 heads at head dims 64, 128, 256; of fewer
// heads, accordingly more tokens) into a ring of three stages, one TMA box of up to 128 rows (tokens x heads) for each page and
// operand; eight compute warps own one kv head each (with fewer heads, a share of its tokens). Both products run on
// m16n8k16 fp16 MMAs with tokens (then dimensions) as the 16 rows and up to 8 query heads as the 8 columns: a tensor
// tile of 128 rows would be 15/16 empty at these group sizes. The codes are widened to fp16 in registers, exactly.
//
// The work of the whole batch is one line of units (tiles), cut into equal stretches, one for each SM, wherever the
// sequences begin and end: ragged batches keep all SMs busy with no knowledge of the lengths on the host. A stretch that
// covers a whole item (request, heads of a CTA) writes the output; one that covers part of it writes its sums to the
// workspace, and paged8_merge_kernel joins the parts in the order of the stretches.
//
// Measured on a B200 (both kernels, device time): 64 requests of 1 - 16381 tokens, 32/8 heads of 128: 167 us for 1.075 GB
// in a replayed graph (6.46 TB/s, 98 % of a plain copy's rate; call by call, with inputs that alternate, 174 - 186 us);
// 4 x 16384 tokens: 33.5 us (4.0 TB/s): 3 us until the first boxes are asked for, 5 - 6 us until the first tile is there (the
// ring of all SMs, 28 MB, is on its way), 1.47 us a tile, up to 3 us between the first and the last SM, 4 us for the merge;
// 1 x 256 tokens: 7.5 us. With one copy loop a warp (cp.async, no producer) the
// first takes 197 us; with two CTAs an SM and half tiles 291 us; with one head a CTA (boxes of 2 KB) 268 us.
#include <cuda.h>

#include <atomic>

#include "fa_paged8.cuh"
#include "fa_sm100.cuh"
#include "fa_tma_host.h"

namespace fa {
namespace {

constexpr int kWarps = 8;                       // compute warps, two groups of four; the first warp of a third group loads
constexpr int kThreads = kWarps * 32 + 128;
constexpr int kStageBytes = 65536;              // K, then V
constexpr int kStages = 3;
constexpr int kMaxCtas = 256;
constexpr int kMergeThreads = 256;
constexpr float kSlack = 10.f;                  // log2 of what a score may pass the softmax reference by
constexpr int kTop = 10;                        // log2 of where a column's largest p * vs is put in fp16's range
constexpr float kRoom = 15.9f;                  // log2 of what p * vs may pass vref by: fp16's largest value, less the error of a log2
constexpr uint32_t kNoPage = 0x7fffbad0u;       // K scale (a NaN of its own) of tokens whose page id is out of range

struct Args {
  int dtype, batch, heads_q, head_dim, group;
  int num_blocks, max_blocks, shift;
  int head_ctas, row_chunks;         // items of a request = groups of heads * chunks of query heads
  int head_shift;                    // log2 of the kv heads of a CTA
  int box_shift, scale_shift;        // log2 of the tokens of a TMA box, of a scale entry (at most 8)
  const void* q;
  int64_t q_sb, q_sh;
  const float* ks;
  const float* vs;
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  const int32_t* table;
  int64_t bt_sb, bt_sk;
  const int32_t* lens;
  int64_t cl_stride;
  void* out;
  int64_t o_sb, o_sh;
  float scale_log2;
  int32_t* status;
  uint32_t poll_limit;  // polls of a barrier wait before it is given up
  int skip_unit;        // test hook: unit of every CTA whose tiles are not brought (-1: none)
  int4* cuts;        // for every CTA: request, item, first CTA and number of CTAs of the item that its stretch begins inside
  float* part_stat;  // (2 * CTAs, rows of a CTA, 2): m, l
  float* part_o;     // (2 * CTAs, rows of a CTA, D)
};

// rows (query heads) that a CTA's items have in the workspace
__host__ __device__ constexpr int item_rows(int heads_per_cta, int nt) { return heads_per_cta * nt * 8; }

template <int D> struct Tile {
  static constexpr int kTokens = 4096 / D;            // tokens of a compute warp in a stage
  static constexpr int kMt = kTokens / 16;            // 16-token tiles
  // A row of shared memory is 128 bytes: a token of one head, of two neighbouring heads of 64 dimensions, or half a token of
  // 256 dimensions (TMA brings rows at one rate whatever their length: 64-byte rows would halve the bandwidth).
  static constexpr int kPair = D == 64 ? 1 : 0;       // log2 of the heads in a row
  static constexpr int kHalves = D == 256 ? 2 : 1;
};

// Rows lie in the 128-byte TMA swizzle: 16-byte chunk c of the row at offset x is chunk c ^ (bits 7 .. 9 of x).
constexpr int kRow = 128;
__device__ __forceinline__ uint32_t swizzle_of(uint32_t x) { return ((x >> 7) & 7u) << 4; }
// token of an MMA row: a permutation (tokens are summed over) with which the K reads (four neighbouring chunks of the rows
// r, r ^ 5) and the V reads (two chunks of four even or four odd rows) of a quarter warp touch every bank once
__device__ __forceinline__ int token_of(int m) { return m ^ ((m & 1) << 2); }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void head_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ int clamped_len(const Args& a, int b) {
  return (int)max((int64_t)0, min((int64_t)a.lens[b * a.cl_stride], (int64_t)a.max_blocks << a.shift));
}

// Units that `len` tokens take. (Lengths go up to 2^31 - 1: here and below, nothing is added to one in 32 bits.)
__device__ __forceinline__ int steps_of(int len, int span) { return (int)(((uint32_t)len + span - 1) / (uint32_t)span); }

// Place in the line of units: request, item of it, step of the item.
struct Cursor {
  int b, item, step, steps, len;
  __device__ __forceinline__ void enter(const Args& a, int span) {
    len = clamped_len(a, b);
    steps = steps_of(len, span);
  }
  __device__ __forceinline__ void advance(const Args& a, int span, int items) {
    if (++step < steps) return;
    step = 0;
    if (++item < items) return;
    item = 0;
    do {
      if (++b >= a.batch) {  // behind the last unit: nothing is read from here
        b = a.batch - 1;
        len = 0;
        return;
      }
      enter(a, span);
    } while (steps == 0);
  }
};

// Stretches: the first `more` CTAs take base + 1 units, the others base.
struct Stretches {
  int64_t base, more;
  __device__ __forceinline__ int64_t begin(int64_t i) const { return i * base + min(i, more); }
  __device__ __forceinline__ int cta_of(int64_t unit) const {
    const int64_t long_part = more * (base + 1);
    return (int)(unit < long_part ? unit / (base + 1) : more + (unit - long_part) / base);
  }
};

template <int D, int NT> struct Smem {
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kScaleStage = Tile<D>::kTokens * kWarps * 8;  // K and V scales of a stage, at one token an entry
  static constexpr int kScales = kStages * kScaleStage;
  static constexpr int kMerge = kWarps * 2048;
  static constexpr int kStats = kWarps * NT * 8 * 8;
  static constexpr int kBytes = kRing + kScales + kMerge + kStats + 1024;  // the ring is moved to a 1024-byte boundary
};

// Waits for a phase, all lanes of a warp alike; a wait that runs out is recorded, and later ones are not begun.
__device__ __forceinline__ void wait_for(uint64_t* bar, uint32_t parity, bool& lost, const Args& a, int code) {
  if (lost) return;
  const bool done = mbar_wait_limit(bar, parity, a.poll_limit);
  lost = __any_sync(0xffffffffu, !done);
  if (lost && a.status != nullptr) *a.status = code;
}

template <typename C8, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    paged8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Args a) {
  using T = Tile<D>;
  constexpr int kTokens = T::kTokens, kMt = T::kMt, kJ = D / 64, kNm = D / 16, kRows = NT * 8;
  constexpr int kRoundTiles = NT == 1 ? 4 : 2, kCols = kRoundTiles * 16;  // columns of a merge round
  constexpr int kHalfBytes = kStageBytes / 2 / T::kHalves;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int64_t scan_s[kWarps];
  __shared__ int64_t start_s[3];
  __shared__ __align__(8) uint64_t full_s[kStages], empty_s[kStages];
  __shared__ int plain_s[kStages];  // whether every token of the stage is there
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads_cta = 1 << a.head_shift, warps_head = kWarps >> a.head_shift;
  const int span = kTokens * warps_head, items = a.head_ctas * a.row_chunks;
  uint8_t* smem = smem_raw + ((1024u - smem_u32(smem_raw)) & 1023u);
  grid_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full_s[i], 33);  // the producer's lanes (scales) and its word that everything is on the way
      mbar_init(&empty_s[i], kWarps);
    }
    mbar_fence_init();
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  grid_dependency_wait();  // nothing above touches global memory: it runs while the kernel before this one ends

  // ---- this CTA's stretch of units
  int64_t total, u_begin, u_end;
  Stretches cut_line;
  {
    const int per = (a.batch + kWarps * 32 - 1) / (kWarps * 32), b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    const int len0 = b0 < b1 ? clamped_len(a, b0) : 0;  // (the only one of this thread up to 256 requests)
    int64_t mine = (int64_t)steps_of(len0, span) * items;
    for (int b = b0 + 1; b < b1; ++b) mine += (int64_t)steps_of(clamped_len(a, b), span) * items;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31 && warp < kWarps) scan_s[warp] = sum;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) sum += scan_s[w];
      total += scan_s[w];
    }
    const int ctas = (int)min((int64_t)gridDim.x, total);
    u_begin = u_end = 0;
    if ((int)blockIdx.x < ctas) {
      if (total <= UINT32_MAX) {
        cut_line.base = (uint32_t)total / (uint32_t)ctas;
      } else {
        cut_line.base = total / ctas;
      }
      cut_line.more = total - cut_line.base * ctas;
      u_begin = cut_line.begin(blockIdx.x);
      u_end = cut_line.begin(blockIdx.x + 1);
    }
    int64_t at = sum - mine;
    if (u_begin < u_end && at <= u_begin && u_begin < sum) {
      for (int b = b0; b < b1; ++b) {
        const int len = b == b0 ? len0 : clamped_len(a, b);
        const int64_t n = (int64_t)steps_of(len, span) * items;
        if (at <= u_begin && u_begin < at + n) {
          start_s[0] = b;
          start_s[1] = at;
          start_s[2] = len;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  const int units = (int)(u_end - u_begin);
  Cursor at;
  if (units > 0) {
    at.b = (int)start_s[0];
    at.len = (int)start_s[2];
    at.steps = steps_of(at.len, span);
    const int64_t rest = u_begin - start_s[1];
    if (rest < INT32_MAX) {
      at.item = (int)rest / at.steps;
      at.step = (int)rest % at.steps;
    } else {
      at.item = (int)(rest / at.steps);
      at.step = (int)(rest % at.steps);
    }
  }
  bool lost = false;

  if (warp >= kWarps) {
    // =============================== producer warp ===============================
    // (the CTA was launched with 168 registers a thread: 56 + 2 * 224 = 3 * 168)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp > kWarps) return;
    const int box = 1 << a.box_shift, boxes = span >> a.box_shift, page_mask = (1 << a.shift) - 1;
    const int entries = (span >> a.scale_shift) << a.head_shift;
    const uint32_t box_bytes = (uint32_t)(box << (a.head_shift - T::kPair)) * kRow;
    auto page_at = [&](const Cursor& c, int off) -> int {  // page of the off-th token of the step
      const int pos0 = c.step * span;
      if (off >= c.len - pos0) return -1;
      const int id = a.table[c.b * a.bt_sb + ((pos0 + off) >> a.shift) * a.bt_sk];
      return id >= 0 && id < a.num_blocks ? id : -1;
    };
    auto fetch = [&](const Cursor& c) -> int { return lane < boxes ? page_at(c, lane * box) : -1; };
    int page = -1;
    if (units > 0) page = fetch(at);
    int stage = 0, issued = 0;
    uint32_t parity = 1;
    for (; issued < units; ++issued) {
      if (issued >= kStages) wait_for(&empty_s[stage], parity, lost, a, 801);
      if (lost) break;
      const int head0 = (at.item / a.row_chunks) << a.head_shift, pos0 = at.step * span;
      uint8_t* kt = smem + stage * kStageBytes;
      const uint32_t st = smem_u32(smem) + Smem<D, NT>::kRing + stage * Smem<D, NT>::kScaleStage;
      if (lane == 0)
        asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full_s[stage])), "n"(kStageBytes) : "memory");
      __syncwarp();
      bool plain = true;
      for (int i = lane; i < boxes && issued != a.skip_unit; i += 32) {
        const int off = i * box, id = i < 32 ? page : page_at(at, off);
        const int in_page = ((pos0 & page_mask) + off) & page_mask;  // (pos0 + off may pass 2^31)
        plain = plain && id >= 0 && off + box <= at.len - pos0;
        // tokens behind the context and pages out of range: a page behind the last one, which reads as zeros
        const int c3 = id >= 0 ? id : a.num_blocks;
#pragma unroll
        for (int h = 0; h < T::kHalves; ++h) {
          tma_load_4d(kt + h * kHalfBytes + i * box_bytes, &k_map, &full_s[stage], h * 128, in_page, head0 >> T::kPair, c3);
          tma_load_4d(kt + kStageBytes / 2 + h * kHalfBytes + i * box_bytes, &v_map, &full_s[stage], h * 128, in_page, head0 >> T::kPair, c3);
        }
      }
      plain = __all_sync(0xffffffffu, plain);
      for (int e0 = 0; e0 < entries; e0 += 32) {
        const int e = e0 + lane, off = (e >> a.head_shift) << a.scale_shift;
        int id = __shfl_sync(0xffffffffu, page, (off >> a.box_shift) & 31);
        if (boxes > 32) id = page_at(at, off);
        if (e >= entries) continue;
        const uint32_t k_to = st + e * 4, v_to = k_to + entries * 4;
        const int head = head0 + (e & (heads_cta - 1));
        if (id >= 0) {
          copy4(k_to, a.ks + id * a.ks_sb + head * a.ks_sh);
          copy4(v_to, a.vs + id * a.vs_sb + head * a.vs_sh);
        } else {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(k_to), "r"(kNoPage) : "memory");
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(v_to), "r"(0) : "memory");
        }
      }
      if (lane == 0) plain_s[stage] = plain;
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_s[stage]);
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_s[stage])) : "memory");
      if (issued + 1 < units) {
        at.advance(a, span, items);
        page = fetch(at);
      }
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
    if (lost) {  // copies on the way land before the CTA leaves
      for (int i = max(0, issued - kStages); i < issued; ++i) {
        bool gone = false;
        wait_for(&full_s[i % kStages], (i / kStages) & 1, gone, a, 802);
      }
    }
    return;
  }

  asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
  // empty contexts have no unit: their rows are zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (clamped_len(a, b) == 0)
      for (int i = tid; i < a.heads_q * (a.head_dim / 2); i += kWarps * 32)
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + b * a.o_sb + (i / (a.head_dim / 2)) * a.o_sh)[i % (a.head_dim / 2)] = 0u;
  if (tid == 0) {
    int4 cut = make_int4(0, 0, 0, 0);
    if (units > 0 && at.step > 0) {
      const int64_t begin = u_begin - at.step;
      const int c0 = cut_line.cta_of(begin), c1 = cut_line.cta_of(begin + at.steps - 1);
      cut = make_int4(at.b, at.item, c0, c1 - c0 + 1);
    }
    a.cuts[blockIdx.x] = cut;
  }

  // =============================== compute warps ===============================
  const int g = lane >> 2, t4 = lane & 3;
  const int wh = warp >> (3 - a.head_shift), wt = warp & (warps_head - 1);
  float* merge = reinterpret_cast<float*>(smem + Smem<D, NT>::kRing + Smem<D, NT>::kScales);
  float2* stats = reinterpret_cast<float2*>(smem + Smem<D, NT>::kRing + Smem<D, NT>::kScales + Smem<D, NT>::kMerge);
  // A box holds its tokens head by head (pair by pair), so token t (of the stage) of head h lies at row
  // (t / box) * box * heads + h * box + t % box: a 16-token tile begins at tile_at[], 8 tokens further is 8 rows inside a
  // box of 16 or more and 8 * heads rows otherwise, and the 8 tokens of a group differ by lane constants.
  const int box = 1 << a.box_shift, layout_shift = a.head_shift - T::kPair;
  const uint32_t step8 = box >= 16 ? 8u * kRow : (uint32_t)(8 << layout_shift) * kRow;
  auto row_of = [&](int t) -> uint32_t { return (uint32_t)(((t >> a.box_shift << a.box_shift) << layout_shift) + (t & (box - 1))) * kRow; };
  uint32_t tile_at[kMt];
#pragma unroll
  for (int mt = 0; mt < kMt; ++mt) tile_at[mt] = row_of(wt * kTokens + mt * 16);
  const uint32_t head_at = smem_u32(smem) + (uint32_t)((wh >> T::kPair) * box) * kRow;
  const uint32_t k_row = row_of(token_of(g)), va_row = row_of(token_of(2 * t4)), vb_row = row_of(token_of(2 * t4 + 1));
  // (the swizzle follows the address: the head's rows count too where a box has fewer than 8 tokens)
  const uint32_t head_rows = (uint32_t)((wh >> T::kPair) * box) * kRow;
  const uint32_t k_swz = swizzle_of(k_row + head_rows), va_swz = swizzle_of(va_row + head_rows), vb_swz = swizzle_of(vb_row + head_rows);
  const uint32_t half_row = (wh & T::kPair) * 4;  // first chunk of the head in its row
  const uint32_t scale8 = (uint32_t)((8 >> a.scale_shift) << a.head_shift) * 4;
  const uint32_t scale_base = smem_u32(smem) + Smem<D, NT>::kRing + wt * kMt * 2 * scale8 +
                              (((token_of(g) >> a.scale_shift) << a.head_shift) + wh) * 4;
  const uint32_t v_scales = (uint32_t)((span >> a.scale_shift) << a.head_shift) * 4;

  uint32_t qf[NT][kJ * 4][2];
  float row_scale[NT][2];       // of rows 2 t4, 2 t4 + 1: softmax scale * log2(e) * the query row's own scale
  float o[NT][kNm][4], m[NT][2], l[NT][2];
  float vinv[NT][2];            // inverses of the powers of two (vref) that the columns' products with V are relative to
  float v_limit = 0.f;          // log2 of this lane's smallest vref, + 127 + kRoom
  int begin_step = 0, stage = 0;
  uint32_t parity = 0;
  for (int u = 0; u < units; ++u) {
    const int head = ((at.item / a.row_chunks) << a.head_shift) + wh, chunk0 = (at.item % a.row_chunks) * kRows;
    if (u == 0 || at.step == 0) {
      // A new item: query rows as fp16 operands. fp16 rows go as they are; a bf16 row is first scaled by the power of
      // two that puts its largest value into [2^14, 2^15), which keeps every bit down to 2^-31 of that value.
      begin_step = at.step;
      v_limit = 1.f + kRoom;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = chunk0 + nt * 8 + g;
        const bool in = r < a.group;
        const int64_t base = at.b * a.q_sb + (int64_t)(head * a.group + (in ? r : 0)) * a.q_sh;
        uint4 raw[kJ][2];
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d = 64 * j + 16 * t4 + 8 * h;
            raw[j][h] = make_uint4(0u, 0u, 0u, 0u);
            if (in && d < a.head_dim)
              raw[j][h] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + base + d);
          }
        float unit = 1.f;
        if (a.dtype == FA_BF16) {
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w[4] = {raw[j][h].x, raw[j][h].y, raw[j][h].z, raw[j][h].w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = DType<__nv_bfloat16>::unpack2(w[i]);
                amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
              }
            }
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          // unit = 2^(exponent - 14), kept normal together with its inverse
          const int e = (int)(__float_as_uint(amax) >> 23) - 14;
          unit = __uint_as_float((uint32_t)min(max(e, 1), 252) << 23);
          const float inverse = __uint_as_float((254u << 23) - __float_as_uint(unit));
#pragma unroll
          for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t* w = reinterpret_cast<uint32_t*>(&raw[j][h]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = DType<__nv_bfloat16>::unpack2(w[i]);
                w[i] = DType<__half>::pack2(f.x * inverse, f.y * inverse);
              }
            }
        }
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          // words of the 16 dimensions 64 j + 16 t4: k-step i multiplies dimensions 4 i .. 4 i + 3 of them
          const uint32_t w[8] = {raw[j][0].x, raw[j][0].y, raw[j][0].z, raw[j][0].w,
                                 raw[j][1].x, raw[j][1].y, raw[j][1].z, raw[j][1].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qf[nt][j * 4 + i][0] = w[2 * i];
            qf[nt][j * 4 + i][1] = w[2 * i + 1];
          }
        }
        const float mine = a.scale_log2 * unit;
        row_scale[nt][0] = __shfl_sync(0xffffffffu, mine, (2 * t4) * 4);
        row_scale[nt][1] = __shfl_sync(0xffffffffu, mine, (2 * t4 + 1) * 4);
        m[nt][0] = m[nt][1] = kNegInf;
        l[nt][0] = l[nt][1] = 0.f;
        vinv[nt][0] = vinv[nt][1] = __uint_as_float(253u << 23);
#pragma unroll
        for (int i = 0; i < kNm; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
      }
    }

    wait_for(&full_s[stage], parity, lost, a, 803);
    const bool plain = plain_s[stage] != 0;
    const uint32_t kt = head_at + stage * kStageBytes, vt = kt + kStageBytes / 2;
    const uint32_t st = scale_base + stage * Smem<D, NT>::kScaleStage;
    const int left = at.len - at.step * span - wt * kTokens;  // tokens of the context from this tile's first on
    if (!lost) {
    // ---- scores: rows are tokens, columns query heads
    float s[kMt][NT][4];
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
      // (256 dimensions are sixteen products in a row with one 16-token tile to work on: four sums instead of one)
      constexpr int kSums = D == 256 ? 4 : 1;
      float sums[kSums][NT][4];
#pragma unroll
      for (int x = 0; x < kSums; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sums[x][nt][c] = 0.f;
      const uint32_t row = kt + tile_at[mt] + k_row;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const uint32_t chunk = (((half_row + t4 + 4 * (j & 1)) << 4) ^ k_swz) + (j >> 1) * kHalfBytes;
        const uint4 ka = lds128(row + chunk), kb = lds128(row + step8 + chunk);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = C8::lo(wa[i]), a1 = C8::lo(wb[i]), a2 = C8::hi(wa[i]), a3 = C8::hi(wb[i]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma(sums[i % kSums][nt], a0, a1, a2, a3, qf[nt][j * 4 + i][0], qf[nt][j * 4 + i][1]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          s[mt][nt][c] = kSums == 1 ? sums[0][nt][c] : (sums[0][nt][c] + sums[1 % kSums][nt][c]) + (sums[2 % kSums][nt][c] + sums[3 % kSums][nt][c]);
    }
    // ---- Scales and mask. m is a reference, not the maximum: it moves (with everything summed so far) only when a score
    // passes it by more than 2^kSlack, so most tiles need no reduction over the warp. The products with V take p * vs
    // relative to a power of two vref, which puts the column's largest p * vs at 2^kTop or above, near the top of fp16's
    // range: a weight keeps its 11 bits down to 2^-24 of the largest, and what is lost lies below 2^-35 of it, so that many
    // tokens of small probability count beside one of a large one. vref follows p * vs, not the scales (a large scale under
    // probabilities next to nothing would push everything else out of the range). Both are looked at again when a score
    // passes m by too much, and when the lane's largest score and largest scale together could leave the range.
    float v_scale[kMt][2], v_most = 0.f;
    float excess = -100.f;  // (so a scale passes vref by less than 2^116, and their ratio stays in fp32)
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
      const uint32_t at0 = st + mt * 2 * scale8, at1 = at0 + scale8;
      const float k0 = lds_f32(at0), k1 = lds_f32(at1);
      v_scale[mt][0] = lds_f32(at0 + v_scales);
      v_scale[mt][1] = lds_f32(at1 + v_scales);
      v_most = fmax3(v_most, fabsf(v_scale[mt][0]), fabsf(v_scale[mt][1]));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[mt][nt][e] *= k0 * row_scale[nt][e];
          s[mt][nt][2 + e] *= k1 * row_scale[nt][e];
        }
      if (!plain) {
        const int r = mt * 16 + token_of(g);
        const bool in0 = r < left && __float_as_uint(k0) != kNoPage, in1 = r + 8 < left && __float_as_uint(k1) != kNoPage;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[mt][nt][e] = in0 ? s[mt][nt][e] : kNegInf;
            s[mt][nt][2 + e] = in1 ? s[mt][nt][2 + e] : kNegInf;
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = kNegInf;
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) top = fmax3(top, s[mt][nt][e], s[mt][nt][2 + e]);
        excess = fmaxf(excess, top - m[nt][e]);  // (-inf) - (-inf) is NaN, which loses
      }
    // (the bits of a positive number, as a number of units of 2^-23, are its log2 + 127 or up to 0.0861 less)
    const bool leaves = excess + __uint2float_rz(__float_as_uint(v_most)) * 0x1p-23f > v_limit;
    if (__any_sync(0xffffffffu, excess > kSlack || leaves)) {
      const float v_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v_most)));
      v_limit = INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = m[nt][e];
#pragma unroll
          for (int mt = 0; mt < kMt; ++mt) top = fmax3(top, s[mt][nt][e], s[mt][nt][2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float z = top == kNegInf ? 0.f : top;
          float w_top = 0.f;  // largest p * vs of the tile
#pragma unroll
          for (int mt = 0; mt < kMt; ++mt)
            w_top = fmax3(w_top, fast_exp2(s[mt][nt][e] - z) * fabsf(v_scale[mt][0]),
                          fast_exp2(s[mt][nt][2 + e] - z) * fabsf(v_scale[mt][1]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, x));
          const float vref_old = __uint_as_float((254u << 23) - __float_as_uint(vinv[nt][e]));
          const float alpha = top == m[nt][e] ? 1.f : fast_exp2(m[nt][e] - top);
          // 2^-kTop of the largest p * vs so far, and never so far below a scale that their ratio leaves fp32
          const float wanted = fmaxf(fmaxf(w_top, alpha * vref_old * (float)(1 << kTop)), 0x1p-100f * v_top);
          const uint32_t ref = (uint32_t)min(max((int)(__float_as_uint(wanted) >> 23) - kTop, 1), 253) << 23;
          const int rise = (int)(__float_as_uint(vref_old) >> 23) - (int)(ref >> 23);
          f[e] = top == m[nt][e] ? __uint_as_float((uint32_t)max(127 + rise, 0) << 23) : fast_exp2(m[nt][e] - top + (float)rise);
          vinv[nt][e] = __uint_as_float((254u << 23) - ref);
          v_limit = fminf(v_limit, (float)(ref >> 23) + kRoom);
          m[nt][e] = top;
          l[nt][e] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < kNm; ++i) {
          o[nt][i][0] *= f[0];
          o[nt][i][1] *= f[1];
          o[nt][i][2] *= f[0];
          o[nt][i][3] *= f[1];
        }
      }
    }
    // ---- probabilities and the products with V: rows are dimensions, columns query heads
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float z0 = m[nt][0] == kNegInf ? 0.f : m[nt][0], z1 = m[nt][1] == kNegInf ? 0.f : m[nt][1];
        const float p00 = fast_exp2(s[mt][nt][0] - z0), p01 = fast_exp2(s[mt][nt][1] - z1);
        const float p10 = fast_exp2(s[mt][nt][2] - z0), p11 = fast_exp2(s[mt][nt][3] - z1);
        l[nt][0] += p00 + p10;
        l[nt][1] += p01 + p11;
        b0[nt] = transpose8x8(DType<__half>::pack2(p00 * (v_scale[mt][0] * vinv[nt][0]), p01 * (v_scale[mt][0] * vinv[nt][1])));
        b1[nt] = transpose8x8(DType<__half>::pack2(p10 * (v_scale[mt][1] * vinv[nt][0]), p11 * (v_scale[mt][1] * vinv[nt][1])));
      }
      auto product = [&](int i, uint32_t wa, uint32_t wb, uint32_t wc, uint32_t wd) {
        // four dimensions of tokens ra, rb (and ra + 8, rb + 8): tiles i (dimensions 0, 1) and i + 1 (2, 3)
        const uint32_t x = __byte_perm(wa, wb, 0x5140), y = __byte_perm(wc, wd, 0x5140);
        const uint32_t z = __byte_perm(wa, wb, 0x7362), w = __byte_perm(wc, wd, 0x7362);
        const uint32_t a0 = C8::lo(x), a1 = C8::hi(x), a2 = C8::lo(y), a3 = C8::hi(y);
        const uint32_t c0 = C8::lo(z), c1 = C8::hi(z), c2 = C8::lo(w), c3 = C8::hi(w);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma(o[nt][i], a0, a1, a2, a3, b0[nt], b1[nt]);
          mma(o[nt][i + 1], c0, c1, c2, c3, b0[nt], b1[nt]);
        }
      };
      // rows behind the context may hold anything, NaN among it: zeros there
      const int r = mt * 16 + token_of(2 * t4), r2 = mt * 16 + token_of(2 * t4 + 1);
      const uint32_t row_a = vt + tile_at[mt] + va_row, row_b = vt + tile_at[mt] + vb_row;
      if constexpr (D == 64) {
        const uint32_t ca = (((half_row + (g >> 1)) << 4) ^ va_swz) + (g & 1) * 8, cb = (((half_row + (g >> 1)) << 4) ^ vb_swz) + (g & 1) * 8;
        uint2 va = lds64(row_a + ca), vb = lds64(row_b + cb);
        uint2 vc = lds64(row_a + step8 + ca), vd = lds64(row_b + step8 + cb);
        if (!plain) {
          if (r >= left) va = make_uint2(0u, 0u);
          if (r2 >= left) vb = make_uint2(0u, 0u);
          if (r + 8 >= left) vc = make_uint2(0u, 0u);
          if (r2 + 8 >= left) vd = make_uint2(0u, 0u);
        }
        product(0, va.x, vb.x, vc.x, vd.x);
        product(2, va.y, vb.y, vc.y, vd.y);
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const uint32_t ca = ((uint32_t)(g << 4) ^ va_swz) + h * kHalfBytes, cb = ((uint32_t)(g << 4) ^ vb_swz) + h * kHalfBytes;
          uint4 va = lds128(row_a + ca), vb = lds128(row_b + cb);
          uint4 vc = lds128(row_a + step8 + ca), vd = lds128(row_b + step8 + cb);
          if (!plain) {
            if (r >= left) va = make_uint4(0u, 0u, 0u, 0u);
            if (r2 >= left) vb = make_uint4(0u, 0u, 0u, 0u);
            if (r + 8 >= left) vc = make_uint4(0u, 0u, 0u, 0u);
            if (r2 + 8 >= left) vd = make_uint4(0u, 0u, 0u, 0u);
          }
          product(8 * h, va.x, vb.x, vc.x, vd.x);
          product(8 * h + 2, va.y, vb.y, vc.y, vd.y);
          product(8 * h + 4, va.z, vb.z, vc.z, vd.z);
          product(8 * h + 6, va.w, vb.w, vc.w, vd.w);
        }
      }
    }
    } else {  // the tile never came: this part of the item hands in nothing
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = kNegInf;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < kNm; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
      }
    }
    __syncwarp();  // every lane is done with the stage
    // A warp that has lost a wait hands no stage back: the loading warp then stops at its own bounded wait, and no barrier
    // is armed again whose phase is still open (arriving there once more is undefined).
    if (lane == 0 && !lost) mbar_arrive(&empty_s[stage]);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }

    // ---- the item ends here, or this CTA's part of it does
    if (at.step + 1 == at.steps || u + 1 == units) {
      const bool whole = begin_step == 0 && at.step + 1 == at.steps;
      const int slot = blockIdx.x * 2 + (begin_step > 0 ? 0 : 1);
      const int rows = item_rows(heads_cta, NT);
      float weight[NT][2], top[NT][2], sum[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
          top[nt][e] = m[nt][e];
          sum[nt][e] = l[nt][e];
          weight[nt][e] = __uint_as_float((254u << 23) - __float_as_uint(vinv[nt][e]));
        }
      if (warps_head > 1) {  // the warps of a head took its tokens by turns
        if (g == 0)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              stats[warp * kRows + nt * 8 + 2 * t4 + e] = make_float2(m[nt][e], l[nt][e]);
        head_barrier(1 + wh, warps_head * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float M = kNegInf, L = 0.f;
            const float2* peer = stats + (warp - wt) * kRows + nt * 8 + 2 * t4 + e;
            for (int w = 0; w < warps_head; ++w) M = fmaxf(M, peer[w * kRows].x);
            const float z = M == kNegInf ? 0.f : M;
            for (int w = 0; w < warps_head; ++w) L += peer[w * kRows].y * fast_exp2(peer[w * kRows].x - z);
            weight[nt][e] *= fast_exp2(m[nt][e] - z);
            top[nt][e] = M;
            sum[nt][e] = L;
          }
      }
      // A whole item is divided by its sum; a part by the sum's power of two, which moves into m (p reaches 2^kSlack, and the
      // sum of many of it times large values would leave fp32).
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (whole) {
            weight[nt][e] = sum[nt][e] == 0.f ? 0.f : weight[nt][e] / sum[nt][e];
          } else {
            const uint32_t power = sum[nt][e] == 0.f ? 127u << 23 : __float_as_uint(sum[nt][e]) & 0x7f800000u;
            const float inverse = __uint_as_float((254u << 23) - power);
            weight[nt][e] *= inverse;
            sum[nt][e] *= inverse;
            top[nt][e] += (float)((int)(power >> 23) - 127);
          }
        }
      if (!whole && wt == 0 && g == 0)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float2*>(a.part_stat + ((int64_t)slot * rows + wh * kRows + nt * 8 + 2 * t4 + e) * 2) =
                make_float2(top[nt][e], sum[nt][e]);
      // four dimensions from d on of one query row
      auto put4 = [&](int row, int d, float4 x) {
        if (chunk0 + row >= a.group || d >= a.head_dim) return;
        if (whole) {
          uint16_t* to = static_cast<uint16_t*>(a.out) + at.b * a.o_sb + (int64_t)(head * a.group + chunk0 + row) * a.o_sh + d;
          *reinterpret_cast<uint2*>(to) = a.dtype == FA_F16
              ? make_uint2(DType<__half>::pack2(x.x, x.y), DType<__half>::pack2(x.z, x.w))
              : make_uint2(DType<__nv_bfloat16>::pack2(x.x, x.y), DType<__nv_bfloat16>::pack2(x.z, x.w));
        } else {
          *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * rows + wh * kRows + row) * D + d) = x;
        }
      };
      constexpr int kPerLane = D == 64 ? 8 : 16;  // neighbouring dimensions of a lane group g
      if (warps_head == 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < kNm; i += 2)
              put4(nt * 8 + 2 * t4 + e, (i / 8) * 128 + kPerLane * g + 2 * (i % 8),
                   make_float4(o[nt][i][e] * weight[nt][e], o[nt][i][2 + e] * weight[nt][e],
                               o[nt][i + 1][e] * weight[nt][e], o[nt][i + 1][2 + e] * weight[nt][e]));
      } else {  // sums of the head's warps, kRoundTiles tiles of dimensions at a time (rolled loops: this code runs once an item)
        float* mine = merge + warp * 512;
#pragma unroll
        for (int round = 0; round < kNm / kRoundTiles; ++round) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < kRoundTiles; ++i) {
                const float* x = o[nt][round * kRoundTiles + i];
                *reinterpret_cast<float2*>(mine + (nt * 8 + 2 * t4 + e) * kCols + g * 2 * kRoundTiles + 2 * i) =
                    make_float2(x[e] * weight[nt][e], x[2 + e] * weight[nt][e]);
              }
          head_barrier(1 + wh, warps_head * 32);
#pragma unroll 1
          for (int x = wt * 32 + lane; x < 128; x += warps_head * 32) {
            const int row = x * 4 / kCols, col = x * 4 % kCols;
            const float* from = merge + (warp - wt) * 512 + x * 4;
            float4 acc = *reinterpret_cast<const float4*>(from);
#pragma unroll 1
            for (int w = 1; w < warps_head; ++w) {
              const float4 y = *reinterpret_cast<const float4*>(from + w * 512);
              acc.x += y.x;
              acc.y += y.y;
              acc.z += y.z;
              acc.w += y.w;
            }
            const int tile = round * kRoundTiles + (col % (2 * kRoundTiles)) / 2;
            put4(row, (tile / 8) * 128 + kPerLane * (col / (2 * kRoundTiles)) + 2 * (tile % 8), acc);
          }
          head_barrier(1 + wh, warps_head * 32);
        }
      }
    }
    if (u + 1 < units) at.advance(a, span, items);
  }
}

// Joins the parts of the items that several CTAs share. A stretch that begins inside an item is one cut of it; an item of
// `parts` stretches has parts - 1 cuts, whose blocks (kMergeSplit a cut) share its rows. With few parts a warp takes a row,
// all of whose parts it loads at once; with many a block does.
constexpr int kMergeSplit = 4;
template <int D, int NT>
__global__ void __launch_bounds__(kMergeThreads) paged8_merge_kernel(const Args a) {
  constexpr int kVec = (D + 127) / 128;
  __shared__ float red_s[kMergeThreads / 32][D];
  __shared__ float2 stat_s[kMergeThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 cut = a.cuts[blockIdx.x + 1];
  const int b = cut.x, item = cut.y, c0 = cut.z, parts = cut.w;
  if (parts == 0) return;
  const int head0 = (item / a.row_chunks) << a.head_shift, chunk0 = (item % a.row_chunks) * NT * 8;
  const int slots = item_rows(1 << a.head_shift, NT);               // rows of a part in the workspace
  const int live = min(NT * 8, a.group - chunk0), rows = live << a.head_shift;  // query heads there are
  const int turn = ((int)blockIdx.x - c0) * kMergeSplit + blockIdx.y, share = (parts - 1) * kMergeSplit;
  auto part_row = [&](int p, int row) {
    return (int64_t)(2 * (c0 + p) + (p == 0 ? 1 : 0)) * slots + (row / live) * NT * 8 + row % live;
  };
  auto store4 = [&](int row, int d, float4 x) {
    uint16_t* to = static_cast<uint16_t*>(a.out) + b * a.o_sb + (int64_t)((head0 + row / live) * a.group + chunk0 + row % live) * a.o_sh + d;
    *reinterpret_cast<uint2*>(to) = a.dtype == FA_F16
        ? make_uint2(DType<__half>::pack2(x.x, x.y), DType<__half>::pack2(x.z, x.w))
        : make_uint2(DType<__nv_bfloat16>::pack2(x.x, x.y), DType<__nv_bfloat16>::pack2(x.z, x.w));
  };

  if (parts <= 8) {
    for (int row = turn + share * warp; row < rows; row += share * (kMergeThreads / 32)) {
      float2 st = make_float2(kNegInf, 0.f);
      if (lane < parts) st = *reinterpret_cast<const float2*>(a.part_stat + part_row(lane, row) * 2);
      float4 x[8][kVec];
#pragma unroll
      for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int c = 0; c < kVec; ++c)
          x[p][c] = *reinterpret_cast<const float4*>(a.part_o + part_row(min(p, parts - 1), row) * D +
                                                     min(lane * 4 + c * 128, a.head_dim - 4));
      float top = st.x;
#pragma unroll
      for (int i = 4; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
      float w = fast_exp2(st.x - (top == kNegInf ? 0.f : top)), sum = w * st.y;
#pragma unroll
      for (int i = 4; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
      w = sum == 0.f ? 0.f : w / sum;
      float4 acc[kVec];
#pragma unroll
      for (int c = 0; c < kVec; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float f = __shfl_sync(0xffffffffu, w, p);  // lanes 0 .. 7 hold the parts' weights
        if (p >= parts) continue;
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
          acc[c].x += f * x[p][c].x;
          acc[c].y += f * x[p][c].y;
          acc[c].z += f * x[p][c].z;
          acc[c].w += f * x[p][c].w;
        }
      }
#pragma unroll
      for (int c = 0; c < kVec; ++c)
        if (lane * 4 + c * 128 < a.head_dim) store4(row, lane * 4 + c * 128, acc[c]);
    }
    return;
  }
  constexpr int kMergeWarps = kMergeThreads / 32;
  for (int row = turn; row < rows; row += share) {
    // warp w joins parts w, w + 8, ...; lane i holds the statistics of the i-th of them
    const int64_t row_at = part_row(1, row) - 2 * slots;  // part p > 0 lies 2 * slots * p behind it, part 0 slots
    auto part_at = [&](int p) { return row_at + (int64_t)(p == 0 ? 1 : 2 * p) * slots; };
    const int mine = warp + kMergeWarps * lane, count = (parts - warp + kMergeWarps - 1) / kMergeWarps;
    float4 x[8][kVec];
    auto load = [&](int i0) {  // (clamped indexes instead of branches: the loads of a batch go out together)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < kVec; ++c)
          x[i][c] = *reinterpret_cast<const float4*>(a.part_o + part_at(warp + kMergeWarps * min(i0 + i, count - 1)) * D +
                                                     min(lane * 4 + c * 128, a.head_dim - 4));
    };
    float2 st = make_float2(kNegInf, 0.f);
    if (mine < parts) st = *reinterpret_cast<const float2*>(a.part_stat + part_at(mine) * 2);
    load(0);
    float top = st.x;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float w = fast_exp2(st.x - (top == kNegInf ? 0.f : top));
    float sum = w * st.y;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    float4 acc[kVec];
#pragma unroll
    for (int c = 0; c < kVec; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < count; i0 += 8) {
      if (i0 > 0) load(i0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = i0 + i < count ? __shfl_sync(0xffffffffu, w, (i0 + i) & 31) : 0.f;
        if (i0 + i >= count) continue;
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
          acc[c].x += f * x[i][c].x;
          acc[c].y += f * x[i][c].y;
          acc[c].z += f * x[i][c].z;
          acc[c].w += f * x[i][c].w;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kVec; ++c)
      if (lane * 4 + c * 128 < D) *reinterpret_cast<float4*>(&red_s[warp][lane * 4 + c * 128]) = acc[c];
    if (lane == 0) stat_s[warp] = make_float2(top, sum);
    __syncthreads();
    if (tid * 4 < a.head_dim) {
      float all = kNegInf, norm = 0.f;
      for (int i = 0; i < kMergeWarps; ++i) all = fmaxf(all, stat_s[i].x);
      if (all == kNegInf) all = 0.f;
      float4 total = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < kMergeWarps; ++i) {
        const float f = fast_exp2(stat_s[i].x - all);
        const float4 y = *reinterpret_cast<const float4*>(&red_s[i][tid * 4]);
        norm += f * stat_s[i].y;
        total.x += f * y.x;
        total.y += f * y.y;
        total.z += f * y.z;
        total.w += f * y.w;
      }
      const float inverse = norm == 0.f ? 0.f : 1.f / norm;
      store4(row, tid * 4, make_float4(total.x * inverse, total.y * inverse, total.z * inverse, total.w * inverse));
    }
    __syncthreads();
  }
}

// How a head layout is cut: padded head dim, query heads an item takes (8 or 16), kv heads a CTA takes.
struct Shape {
  int D, nt, head_shift, row_chunks, box_shift;
};
Shape shape_of(const fa_paged8_params& p) {
  Shape s;
  const int group = p.heads_q / p.heads_kv;
  s.head_shift = 3;
  while (p.heads_kv % (1 << s.head_shift)) --s.head_shift;
  // Two neighbouring heads of 64 dimensions make a row (see Tile); where they are not neighbours, and for fewer dimensions,
  // rows are padded to 128 by the tensor map (which reads nothing for the padding).
  const bool pairs = p.head_dim == 64 && s.head_shift > 0 && p.k_strides[2] == 64 && p.v_strides[2] == 64;
  s.D = pairs ? 64 : p.head_dim <= 128 ? 128 : 256;
  // A box is up to 128 rows (16 KB) of a page: boxes of 16 rows reach 60 % of the rate of boxes of 64 and more.
  const int layout_shift = s.head_shift - (pairs ? 1 : 0);
  s.box_shift = 0;
  while ((2 << s.box_shift) <= p.block_size && (2 << s.box_shift << layout_shift) <= 128) ++s.box_shift;
  s.nt = group > 8 && s.D <= 128 ? 2 : 1;
  s.row_chunks = (group + s.nt * 8 - 1) / (s.nt * 8);
  return s;
}

// What the host asks the driver once per device (the answers cannot change): a call costs about half a microsecond.
constexpr int kMaxDevices = 64;
int current_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) return dev;
  cudaGetLastError();
  return -1;
}
int cta_count() {
  static std::atomic<int> known[kMaxDevices];
  const int dev = current_device();
  if (dev >= 0 && dev < kMaxDevices && known[dev].load(std::memory_order_relaxed) > 0) return known[dev].load(std::memory_order_relaxed);
  int sms = 0;
  if (dev < 0 || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    cudaGetLastError();
    return set_error(FA_ERR_DEVICE, "cannot query the SM count of the current device");
  }
  sms = sms < kMaxCtas ? sms : kMaxCtas;
  if (dev < kMaxDevices) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// (dim, token of the page, head, page) with a box of one row's bytes x a box's tokens x a CTA's heads
int make_cache_map(CUtensorMap* map, const void* ptr, const fa_paged8_params& p, const int64_t (&st)[4], const Shape& s) {
  TensorMapEncodeFn enc = tensor_map_encoder();
  if (enc == nullptr) return set_error(FA_ERR_DEVICE, "cuTensorMapEncodeTiled is not available from this driver");
  const int pair = s.D == 64 ? 1 : 0, heads = p.heads_kv >> pair;
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim << pair, (cuuint64_t)p.block_size, (cuuint64_t)heads, (cuuint64_t)p.num_blocks};
  auto stride = [&](int64_t x, int64_t n) { return (cuuint64_t)(n > 1 ? x : 256); };  // a size-1 dimension never advances
  const cuuint64_t strides[3] = {stride(st[1], p.block_size), stride(st[2] << pair, heads), stride(st[0], p.num_blocks)};
  const cuuint32_t box[4] = {kRow, 1u << s.box_shift, 1u << (s.head_shift - pair), 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FA_ERR_UNSUPPORTED, "8-bit paged decode: no tensor map for this cache layout (code %d)", (int)r);
  return 0;
}

template <typename C8, int D, int NT>
int launch(const CUtensorMap& k, const CUtensorMap& v, const Args& a, int ctas, cudaStream_t stream) {
  auto kernel = paged8_kernel<C8, D, NT>;
  constexpr int smem = Smem<D, NT>::kBytes;
  static_assert(smem <= 227 * 1024 - 512, "shared memory of an SM");
  static std::atomic<bool> prepared[kMaxDevices];
  const int dev = current_device();
  cudaError_t e = cudaSuccess;
  if (dev < 0 || dev >= kMaxDevices || !prepared[dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev >= 0 && dev < kMaxDevices) prepared[dev].store(true, std::memory_order_relaxed);
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, k, v, a);
  if (e == cudaSuccess && ctas > 1) {
    cfg.gridDim = dim3(ctas - 1, kMergeSplit);
    cfg.blockDim = dim3(kMergeThreads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged8_merge_kernel<D, NT>, a);
  }
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return set_error(FA_ERR_LAUNCH, "8-bit paged decode launch failed: %s", cudaGetErrorString(e));
}

template <typename C8>
int dispatch(const Shape& s, const CUtensorMap& k, const CUtensorMap& v, const Args& a, int ctas, cudaStream_t stream) {
  if (s.D == 64) return s.nt == 1 ? launch<C8, 64, 1>(k, v, a, ctas, stream) : launch<C8, 64, 2>(k, v, a, ctas, stream);
  if (s.D == 128) return s.nt == 1 ? launch<C8, 128, 1>(k, v, a, ctas, stream) : launch<C8, 128, 2>(k, v, a, ctas, stream);
  return launch<C8, 256, 1>(k, v, a, ctas, stream);
}

}  // namespace

int64_t paged8_workspace_bytes(const fa_paged8_params& p) {
  const int ctas = cta_count();
  if (ctas < 0) return ctas;
  const Shape s = shape_of(p);
  return (int64_t)ctas * sizeof(int4) + (int64_t)2 * ctas * item_rows(1 << s.head_shift, s.nt) * (s.D + 2) * 4;
}

int launch_decode_paged8(const fa_paged8_params& p, cudaStream_t stream) {
  const int ctas = cta_count();
  if (ctas < 0) return ctas;
  const Shape s = shape_of(p);
  if (((int64_t)p.max_blocks * p.block_size) > INT32_MAX)
    return set_error(FA_ERR_UNSUPPORTED, "8-bit paged decode: a block table of more than 2^31 - 1 tokens");
  CUtensorMap k, v;
  int rc = make_cache_map(&k, p.k_cache, p, p.k_strides, s);
  if (!rc) rc = make_cache_map(&v, p.v_cache, p, p.v_strides, s);
  if (rc) return rc;
  Args a = {};
  a.dtype = p.dtype;
  a.batch = p.batch;
  a.heads_q = p.heads_q;
  a.head_dim = p.head_dim;
  a.group = p.heads_q / p.heads_kv;
  a.num_blocks = p.num_blocks;
  a.max_blocks = p.max_blocks;
  while ((1 << a.shift) < p.block_size) ++a.shift;
  a.head_shift = s.head_shift;
  a.head_ctas = p.heads_kv >> s.head_shift;
  a.row_chunks = s.row_chunks;
  a.box_shift = s.box_shift;
  a.scale_shift = s.box_shift < 3 ? s.box_shift : 3;
  a.q = p.q;
  a.q_sb = p.q_strides[0];
  a.q_sh = p.q_strides[1];
  a.ks = p.k_scales;
  a.vs = p.v_scales;
  a.ks_sb = p.ks_strides[0];
  a.ks_sh = p.ks_strides[1];
  a.vs_sb = p.vs_strides[0];
  a.vs_sh = p.vs_strides[1];
  a.table = p.block_table;
  a.bt_sb = p.bt_strides[0];
  a.bt_sk = p.bt_strides[1];
  a.lens = p.context_lens;
  a.cl_stride = p.cl_stride;
  a.out = p.out;
  a.o_sb = p.o_strides[0];
  a.o_sh = p.o_strides[1];
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.status = p.status;
  take_decode_fault_injection(&a.poll_limit, &a.skip_unit);
  a.cuts = static_cast<int4*>(p.workspace);
  a.part_stat = reinterpret_cast<float*>(a.cuts + ctas);
  a.part_o = a.part_stat + (int64_t)2 * ctas * item_rows(1 << s.head_shift, s.nt) * 2;
  return p.cache_dtype == FA_CACHE_E4M3 ? dispatch<CodeE4M3>(s, k, v, a, ctas, stream)
                                        : dispatch<CodeInt8>(s, k, v, a, ctas, stream);
}

}  // namespace fa
