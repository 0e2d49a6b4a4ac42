// Decode attention over a paged 8-bit cache (fa_decode_paged8).
//
//   o = sum_t p_t vs_t v_t / sum_t p_t,   p_t = 2^(s_t - m),   s_t = log2(e) * softmax_scale * ks_t * (q . k_t)
//
// with ks_t, vs_t the scales of the page that holds token t. One pass over the cache with running m and sums; every byte
// is read once for all query heads of its kv head, so the bound is HBM: 2 * head_dim bytes a token and kv head.
//
// A warp owns one kv head and streams tiles of 8 KB (64, 32 or 16 tokens of K and V at head dims 64, 128, 256) through a
// ring of its own in shared memory, filled with cp.async; no warp waits for another inside the loop. Both products run on
// m16n8k16 fp16 MMAs with tokens (then dimensions) as the 16 rows and up to 8 query heads as the 8 columns: a tensor
// tile of 128 rows would be 15/16 empty at these group sizes. The codes are widened to fp16 in registers, exactly.
//
// The work of the whole batch is one line of units (a tile for every warp of the CTA), cut into equal stretches, one for
// each SM, wherever the sequences begin and end: ragged batches keep all SMs busy with no knowledge of the lengths on the
// host. A stretch that covers a whole item (request, heads of a CTA) writes the output; one that covers part of it writes
// its sums to the workspace, and paged8_merge_kernel joins the parts in the order of the stretches.
#include "fa_paged8.cuh"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTileBytes = 8192;  // K and V of one warp's tile
constexpr int kStages = 3;
constexpr int kMaxCtas = 256;

struct Args {
  int dtype, batch, heads_q, heads_kv, head_dim, group;
  int num_blocks, max_blocks, shift;
  int head_ctas, row_chunks, warps_per_head;  // items of a request = heads_kv / heads a CTA * chunks of query heads
  const void* q;
  int64_t q_sb, q_sh;
  const uint8_t* k;
  const uint8_t* v;
  uint32_t k_sb, k_st, v_sb, v_st;  // bytes
  int64_t k_sh, v_sh;
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
  int64_t* prefix;   // batch + 1: first unit of every request
  float* part_stat;  // (2 * CTAs, rows of a CTA, 2): m, l
  float* part_o;     // (2 * CTAs, rows of a CTA, D)
};

// rows (query heads) that a CTA's items have in the workspace
__host__ __device__ constexpr int item_rows(int heads_per_cta, int nt) { return heads_per_cta * nt * 8; }

template <int D> struct Tile {
  static constexpr int kTokens = kTileBytes / (2 * D);
  static constexpr int kMt = kTokens / 16;            // 16-token tiles
  static constexpr int kPages = kTokens > 32 ? 2 : 1; // page ids that a lane holds
  static constexpr int kLanes = D / 16;               // lanes a row in a 16-byte copy
};

// Byte offset of a 16-byte chunk of a row. The XOR spreads both access patterns over the banks: K reads four neighbouring
// chunks of the rows r and r ^ 5, V two neighbouring chunks of four even (or four odd) rows.
template <int D>
__device__ __forceinline__ int chunk_at(int row, int chunk) {
  return row * D + ((D == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) << 4);
}
// token of an MMA row: a permutation that makes the reads above free of bank conflicts (tokens are summed over)
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
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
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
// copies of `bytes` (0 or all) with the rest zero: rows that are not there become zeros, NaN patterns behind a context
// never reach the products
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void head_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ int clamped_len(const Args& a, int b) {
  return (int)max((int64_t)0, min((int64_t)a.lens[b * a.cl_stride], (int64_t)a.max_blocks << a.shift));
}

// Place in the line of units: request, item of it, step of the item.
struct Cursor {
  int b, item, step, steps, len;
  __device__ __forceinline__ void enter(const Args& a, int span) {
    len = clamped_len(a, b);
    steps = (len + span - 1) / span;
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

template <int D, int NT> struct Smem {
  static constexpr int kRing = kWarps * kStages * kTileBytes;
  static constexpr int kScaleStage = Tile<D>::kTokens * 8 + 8;  // K scales, V scales, two mask words
  static constexpr int kScales = kWarps * kStages * kScaleStage;
  static constexpr int kMerge = kWarps * 2048;
  static constexpr int kStats = kWarps * NT * 8 * 16;
  static constexpr int kBytes = kRing + kScales + kMerge + kStats;
};

template <typename C8, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1) paged8_kernel(const Args a) {
  using T = Tile<D>;
  constexpr int kTokens = T::kTokens, kMt = T::kMt, kJ = D / 64, kNm = D / 16, kRows = NT * 8;
  constexpr int kRoundTiles = NT == 1 ? 4 : 2, kCols = kRoundTiles * 16;  // columns of a merge round
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan_s[kWarps + 1];
  __shared__ int64_t start_s[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int heads_cta = kWarps / a.warps_per_head, wh = warp / a.warps_per_head, wt = warp % a.warps_per_head;
  const int span = kTokens * a.warps_per_head, items = a.head_ctas * a.row_chunks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's stretch of units
  int64_t total, u_begin, u_end;
  int ctas;
  {
    const int per = (a.batch + kThreads - 1) / kThreads, b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += (int64_t)((clamped_len(a, b) + span - 1) / span) * items;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) scan_s[warp] = sum;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) sum += scan_s[w];
      total += scan_s[w];
    }
    ctas = (int)min((int64_t)gridDim.x, total);
    u_begin = u_end = 0;
    if ((int)blockIdx.x < ctas) {
      u_begin = blockIdx.x * total / ctas;
      u_end = (blockIdx.x + 1) * total / ctas;
    }
    int64_t at = sum - mine;
    const bool here = mine > 0 && at <= u_begin && u_begin < sum;
    if (here || blockIdx.x == 0) {
      for (int b = b0; b < b1; ++b) {
        const int64_t n = (int64_t)((clamped_len(a, b) + span - 1) / span) * items;
        if (blockIdx.x == 0) a.prefix[b] = at;
        if (here && at <= u_begin && u_begin < at + n) {
          start_s[0] = b;
          start_s[1] = at;
        }
        at += n;
      }
    }
    if (blockIdx.x == 0 && tid == 0) a.prefix[a.batch] = total;
    __syncthreads();
  }
  // empty contexts have no unit: their rows are zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (clamped_len(a, b) == 0)
      for (int i = tid; i < a.heads_q * (a.head_dim / 2); i += kThreads)
        reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + b * a.o_sb + (i / (a.head_dim / 2)) * a.o_sh)[i % (a.head_dim / 2)] = 0u;
  if (u_begin == u_end) return;

  const uint32_t ring = smem_u32(smem) + warp * kStages * kTileBytes;
  const uint32_t scales = smem_u32(smem) + Smem<D, NT>::kRing + warp * kStages * Smem<D, NT>::kScaleStage;
  float* merge = reinterpret_cast<float*>(smem + Smem<D, NT>::kRing + Smem<D, NT>::kScales);
  float4* stats = reinterpret_cast<float4*>(smem + Smem<D, NT>::kRing + Smem<D, NT>::kScales + Smem<D, NT>::kMerge);

  Cursor put;
  put.b = (int)start_s[0];
  put.enter(a, span);
  {
    const int64_t rest = u_begin - start_s[1];
    put.item = (int)(rest / put.steps);
    put.step = (int)(rest % put.steps);
  }
  Cursor get = put;
  const int units = (int)(u_end - u_begin);

  // ---- producer side: page ids of the next tile are fetched one tile ahead of its copies
  int page[T::kPages];
  auto fetch_pages = [&]() {
#pragma unroll
    for (int i = 0; i < T::kPages; ++i) {
      const int pos = put.step * span + wt * kTokens + lane + 32 * i;
      page[i] = -1;
      if (pos < put.len && lane + 32 * i < kTokens) {
        const int id = a.table[put.b * a.bt_sb + (pos >> a.shift) * a.bt_sk];
        if (id >= 0 && id < a.num_blocks) page[i] = id;
      }
    }
  };
  auto issue = [&](int stage) {
    const int head = (put.item / a.row_chunks) * heads_cta + wh;
    const uint32_t kt = ring + stage * kTileBytes, vt = kt + kTileBytes / 2;
    const uint32_t st = scales + stage * Smem<D, NT>::kScaleStage;
    uint32_t mask[T::kPages];
#pragma unroll
    for (int i = 0; i < T::kPages; ++i) {
      mask[i] = __ballot_sync(0xffffffffu, page[i] >= 0);
      const int64_t id = max(page[i], 0);
      const int bytes = page[i] >= 0 ? 4 : 0;
      if (lane + 32 * i < kTokens) {
        copy4(st + (lane + 32 * i) * 4, a.ks + id * a.ks_sb + head * a.ks_sh, bytes);
        copy4(st + (kTokens + lane + 32 * i) * 4, a.vs + id * a.vs_sb + head * a.vs_sh, bytes);
      }
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(st + kTokens * 8 + i * 4), "r"(mask[i]) : "memory");
    }
    const int row0 = lane / T::kLanes, chunk = lane % T::kLanes;
    const uint8_t* kh = a.k + head * a.k_sh + chunk * 16;
    const uint8_t* vh = a.v + head * a.v_sh + chunk * 16;
    const uint32_t within = (1u << a.shift) - 1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int tok = j * (32 / T::kLanes) + row0;
      const int i = j * (32 / T::kLanes) / 32;
      const uint32_t id = max(__shfl_sync(0xffffffffu, page[i], tok & 31), 0);
      const uint32_t in_page = (put.step * span + wt * kTokens + tok) & within;
      const int bytes = ((mask[i] >> (tok & 31)) & 1) && chunk * 16 < a.head_dim ? 16 : 0;
      const int at = chunk_at<D>(tok, chunk);
      copy16(kt + at, kh + (uint64_t)id * a.k_sb + (uint64_t)in_page * a.k_st, bytes);
      copy16(vt + at, vh + (uint64_t)id * a.v_sb + (uint64_t)in_page * a.v_st, bytes);
    }
  };
  int put_left = units;
  auto produce = [&](int stage) {
    if (put_left > 0) {
      issue(stage);
      if (--put_left > 0) {
        put.advance(a, span, items);
        fetch_pages();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch_pages();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) produce(s);

  // ---- consumer side
  uint32_t qf[NT][kJ * 4][2];
  float row_scale[NT][2];       // of rows 2 t4, 2 t4 + 1: softmax scale * log2(e) * the query row's own scale
  float o[NT][kNm][4], m[NT][2], l[NT][2];
  float vref = 0.f;             // power of two that the products with V are relative to
  int begin_step = 0;

  int stage = 0, fill = kStages - 1;
  for (int u = 0; u < units; ++u) {
    const int head = (get.item / a.row_chunks) * heads_cta + wh, chunk0 = (get.item % a.row_chunks) * kRows;
    if (u == 0 || get.step == 0) {
      // A new item: query rows as fp16 operands. fp16 rows go as they are; a bf16 row is first scaled by the power of
      // two that puts its largest value into [2^14, 2^15), which keeps every bit down to 2^-28 of that value.
      begin_step = get.step;
      vref = __uint_as_float(1u << 23);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = chunk0 + nt * 8 + g;
        const bool in = r < a.group;
        const int64_t base = get.b * a.q_sb + (int64_t)(head * a.group + (in ? r : 0)) * a.q_sh;
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
#pragma unroll
        for (int i = 0; i < kNm; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
      }
    }

    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    produce(fill);
    fill = fill + 1 == kStages ? 0 : fill + 1;

    const uint32_t kt = ring + stage * kTileBytes, vt = kt + kTileBytes / 2;
    const uint32_t st = scales + stage * Smem<D, NT>::kScaleStage;
    // ---- scores: rows are tokens, columns query heads
    float s[kMt][NT][4];
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[mt][nt][c] = 0.f;
      const int r = mt * 16 + token_of(g);
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const uint4 ka = lds128(kt + chunk_at<D>(r, t4 + 4 * j)), kb = lds128(kt + chunk_at<D>(r + 8, t4 + 4 * j));
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = C8::lo(wa[i]), a1 = C8::lo(wb[i]), a2 = C8::hi(wa[i]), a3 = C8::hi(wb[i]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma(s[mt][nt], a0, a1, a2, a3, qf[nt][j * 4 + i][0], qf[nt][j * 4 + i][1]);
        }
      }
    }
    // ---- scales, mask, running maximum
    float m_new[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m_new[nt][0] = m[nt][0], m_new[nt][1] = m[nt][1];
    float v_scale[kMt][2];
    uint32_t v_top = 0u;
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
      const int r = mt * 16 + token_of(g);
      float k0, k1;
      uint32_t mask;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(k0) : "r"(st + r * 4));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(k1) : "r"(st + (r + 8) * 4));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v_scale[mt][0]) : "r"(st + (kTokens + r) * 4));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v_scale[mt][1]) : "r"(st + (kTokens + r + 8) * 4));
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(mask) : "r"(st + kTokens * 8 + (mt / 2) * 4));
      const bool in0 = (mask >> (r & 31)) & 1, in1 = (mask >> ((r + 8) & 31)) & 1;
      v_top = max(v_top, max(__float_as_uint(v_scale[mt][0]) & 0x7fffffffu, __float_as_uint(v_scale[mt][1]) & 0x7fffffffu));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[mt][nt][e];
          float& y = s[mt][nt][2 + e];
          x = in0 ? x * (k0 * row_scale[nt][e]) : kNegInf;
          y = in1 ? y * (k1 * row_scale[nt][e]) : kNegInf;
          m_new[nt][e] = fmax3(m_new[nt][e], x, y);
        }
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) m_new[nt][e] = fmaxf(m_new[nt][e], __shfl_xor_sync(0xffffffffu, m_new[nt][e], x));
    // ---- The products with V take p * vs relative to the largest |vs| so far (its power of two), so that they are fp16
    // numbers near 1 whatever the pages' scales: rounding them costs 2^-11 of each, 2^-25 of the unit when they are tiny.
    v_top = min(__reduce_max_sync(0xffffffffu, v_top) & 0x7f800000u, 0x7e800000u);
    const float vref_new = fmaxf(vref, __uint_as_float(v_top));
    const float v_inv = __uint_as_float((254u << 23) - __float_as_uint(vref_new));
    bool moved = vref_new != vref;
    float alpha[NT][2];
    const float v_alpha = vref * v_inv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        moved = moved || m_new[nt][e] != m[nt][e];
        m[nt][e] = m[nt][e] == m_new[nt][e] ? 0.f : m[nt][e] - m_new[nt][e];
        alpha[nt][e] = fast_exp2(m[nt][e]);
        m[nt][e] = m_new[nt][e];
        l[nt][e] *= alpha[nt][e];
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = alpha[nt][0] * v_alpha, f1 = alpha[nt][1] * v_alpha;
#pragma unroll
        for (int i = 0; i < kNm; ++i) {
          o[nt][i][0] *= f0;
          o[nt][i][1] *= f1;
          o[nt][i][2] *= f0;
          o[nt][i][3] *= f1;
        }
      }
    }
    vref = vref_new;
    // ---- probabilities and the products with V: rows are dimensions, columns query heads
#pragma unroll
    for (int mt = 0; mt < kMt; ++mt) {
      uint32_t b0[NT], b1[NT];
      const float v0 = v_scale[mt][0] * v_inv, v1 = v_scale[mt][1] * v_inv;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float z0 = m[nt][0] == kNegInf ? 0.f : m[nt][0], z1 = m[nt][1] == kNegInf ? 0.f : m[nt][1];
        const float p00 = fast_exp2(s[mt][nt][0] - z0), p01 = fast_exp2(s[mt][nt][1] - z1);
        const float p10 = fast_exp2(s[mt][nt][2] - z0), p11 = fast_exp2(s[mt][nt][3] - z1);
        l[nt][0] += p00 + p10;
        l[nt][1] += p01 + p11;
        b0[nt] = transpose8x8(DType<__half>::pack2(p00 * v0, p01 * v0));
        b1[nt] = transpose8x8(DType<__half>::pack2(p10 * v1, p11 * v1));
      }
      const int ra = mt * 16 + token_of(2 * t4), rb = mt * 16 + token_of(2 * t4 + 1);
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
      if constexpr (D == 64) {
        const int at = (g & 1) * 8;
        const uint2 va = lds64(vt + chunk_at<D>(ra, g >> 1) + at), vb = lds64(vt + chunk_at<D>(rb, g >> 1) + at);
        const uint2 vc = lds64(vt + chunk_at<D>(ra + 8, g >> 1) + at), vd = lds64(vt + chunk_at<D>(rb + 8, g >> 1) + at);
        product(0, va.x, vb.x, vc.x, vd.x);
        product(2, va.y, vb.y, vc.y, vd.y);
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const uint4 va = lds128(vt + chunk_at<D>(ra, g + 8 * h)), vb = lds128(vt + chunk_at<D>(rb, g + 8 * h));
          const uint4 vc = lds128(vt + chunk_at<D>(ra + 8, g + 8 * h)), vd = lds128(vt + chunk_at<D>(rb + 8, g + 8 * h));
          product(8 * h, va.x, vb.x, vc.x, vd.x);
          product(8 * h + 2, va.y, vb.y, vc.y, vd.y);
          product(8 * h + 4, va.z, vb.z, vc.z, vd.z);
          product(8 * h + 6, va.w, vb.w, vc.w, vd.w);
        }
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;

    // ---- the item ends here, or this CTA's part of it does
    if (get.step + 1 == get.steps || u + 1 == units) {
      const bool whole = begin_step == 0 && get.step + 1 == get.steps;
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
          weight[nt][e] = vref;
        }
      if (a.warps_per_head > 1) {  // the warps of a head took its tokens by turns
        if (g == 0)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              stats[warp * kRows + nt * 8 + 2 * t4 + e] = make_float4(m[nt][e], l[nt][e], 0.f, 0.f);
        head_barrier(1 + wh, a.warps_per_head * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float M = kNegInf, L = 0.f;
            const float4* at = stats + (warp - wt) * kRows + nt * 8 + 2 * t4 + e;
            for (int w = 0; w < a.warps_per_head; ++w) M = fmaxf(M, at[w * kRows].x);
            const float z = M == kNegInf ? 0.f : M;
            for (int w = 0; w < a.warps_per_head; ++w) L += at[w * kRows].y * fast_exp2(at[w * kRows].x - z);
            weight[nt][e] = vref * fast_exp2(m[nt][e] - z);
            top[nt][e] = M;
            sum[nt][e] = L;
          }
      }
      if (whole)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) weight[nt][e] = sum[nt][e] == 0.f ? 0.f : weight[nt][e] / sum[nt][e];
      else if (wt == 0 && g == 0)
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
          uint16_t* to = static_cast<uint16_t*>(a.out) + get.b * a.o_sb + (int64_t)(head * a.group + chunk0 + row) * a.o_sh + d;
          *reinterpret_cast<uint2*>(to) = a.dtype == FA_F16
              ? make_uint2(DType<__half>::pack2(x.x, x.y), DType<__half>::pack2(x.z, x.w))
              : make_uint2(DType<__nv_bfloat16>::pack2(x.x, x.y), DType<__nv_bfloat16>::pack2(x.z, x.w));
        } else {
          *reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * rows + wh * kRows + row) * D + d) = x;
        }
      };
      constexpr int kPerLane = D == 64 ? 8 : 16;  // neighbouring dimensions of a lane group g
      if (a.warps_per_head == 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < kNm; i += 2)
              put4(nt * 8 + 2 * t4 + e, (i / 8) * 128 + kPerLane * g + 2 * (i % 8),
                   make_float4(o[nt][i][e] * weight[nt][e], o[nt][i][2 + e] * weight[nt][e],
                               o[nt][i + 1][e] * weight[nt][e], o[nt][i + 1][2 + e] * weight[nt][e]));
      } else {
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
          head_barrier(1 + wh, a.warps_per_head * 32);
          for (int x = wt * 32 + lane; x < 128; x += a.warps_per_head * 32) {
            const int row = x * 4 / kCols, col = x * 4 % kCols;
            const float* from = merge + (warp - wt) * 512 + x * 4;
            float4 acc = *reinterpret_cast<const float4*>(from);
            for (int w = 1; w < a.warps_per_head; ++w) {
              const float4 y = *reinterpret_cast<const float4*>(from + w * 512);
              acc.x += y.x;
              acc.y += y.y;
              acc.z += y.z;
              acc.w += y.w;
            }
            const int tile = round * kRoundTiles + (col % (2 * kRoundTiles)) / 2;
            put4(row, (tile / 8) * 128 + kPerLane * (col / (2 * kRoundTiles)) + 2 * (tile % 8), acc);
          }
          head_barrier(1 + wh, a.warps_per_head * 32);
        }
      }
    }
    if (u + 1 < units) get.advance(a, span, items);
    __syncwarp();  // every lane is done with the stage before it is filled again
  }
}

// Joins the parts of the items that several CTAs share. The boundary between the stretches of CTAs i - 1 and i lies inside
// at most one item; an item of `parts` stretches has parts - 1 boundaries, and their blocks share its rows.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) paged8_merge_kernel(const Args a, int grid_ctas) {
  __shared__ float weight_s[kMaxCtas];
  __shared__ float red_s[kWarps][D];
  __shared__ float part_s[kWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t total = a.prefix[a.batch];
  const int64_t ctas = min((int64_t)grid_ctas, total);
  const int boundary = blockIdx.x + 1;
  if (boundary >= ctas) return;
  const int64_t u = boundary * total / ctas;
  int lo = 0, hi = a.batch - 1;  // the last request that starts at or before u (requests without units start there too)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.prefix[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo, items = a.head_ctas * a.row_chunks;
  const int64_t first = a.prefix[b], steps = (a.prefix[b + 1] - first) / items;
  const int item = (int)((u - first) / steps);
  const int64_t begin = first + item * steps;
  if (begin == u) return;
  const int c0 = (int)(((begin + 1) * ctas - 1) / total), c1 = (int)(((begin + steps) * ctas - 1) / total);
  const int parts = c1 - c0 + 1, share = parts - 1;
  const int heads_cta = kWarps / a.warps_per_head, rows = item_rows(heads_cta, NT);
  const int head0 = (item / a.row_chunks) * heads_cta, chunk0 = (item % a.row_chunks) * NT * 8;
  auto part_row = [&](int p, int row) { return ((int64_t)(2 * (c0 + p) + (p == 0 ? 1 : 0)) * rows + row); };
  auto store4 = [&](int row, int d, float4 x) {
    uint16_t* to = static_cast<uint16_t*>(a.out) + b * a.o_sb +
                   (int64_t)((head0 + row / (NT * 8)) * a.group + chunk0 + row % (NT * 8)) * a.o_sh + d;
    *reinterpret_cast<uint2*>(to) = a.dtype == FA_F16
        ? make_uint2(DType<__half>::pack2(x.x, x.y), DType<__half>::pack2(x.z, x.w))
        : make_uint2(DType<__nv_bfloat16>::pack2(x.x, x.y), DType<__nv_bfloat16>::pack2(x.z, x.w));
  };
  auto is_row = [&](int row) { return row < rows && chunk0 + row % (NT * 8) < a.group; };
  const int turn = boundary - c0 - 1;

  if (parts <= 8) {  // few parts: a warp takes a row
    for (int row = turn + share * warp; row < rows; row += share * kWarps) {
      if (!is_row(row)) continue;
      float2 st = make_float2(kNegInf, 0.f);
      if (lane < parts) st = *reinterpret_cast<const float2*>(a.part_stat + part_row(lane, row) * 2);
      float top = st.x;
#pragma unroll
      for (int x = 4; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      float w = fast_exp2(st.x - (top == kNegInf ? 0.f : top)), sum = w * st.y;
#pragma unroll
      for (int x = 4; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      w = sum == 0.f ? 0.f : w / sum;
      float4 acc[(D + 127) / 128];
#pragma unroll
      for (int c = 0; c < (D + 127) / 128; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = 0; p < parts; ++p) {
        const float f = __shfl_sync(0xffffffffu, w, p);  // lanes 0 .. 7 hold the parts' weights
#pragma unroll
        for (int c = 0; c < (D + 127) / 128; ++c) {
          const int d = lane * 4 + c * 128;
          if (d >= a.head_dim) continue;
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + part_row(p, row) * D + d);
          acc[c].x += f * x.x;
          acc[c].y += f * x.y;
          acc[c].z += f * x.z;
          acc[c].w += f * x.w;
        }
      }
#pragma unroll
      for (int c = 0; c < (D + 127) / 128; ++c)
        if (lane * 4 + c * 128 < a.head_dim) store4(row, lane * 4 + c * 128, acc[c]);
    }
    return;
  }
  for (int row = turn; row < rows; row += share) {  // many parts: the block takes a row
    if (!is_row(row)) continue;
    float2 st = make_float2(kNegInf, 0.f);
    if (tid < parts) st = *reinterpret_cast<const float2*>(a.part_stat + part_row(tid, row) * 2);
    float top = st.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    __syncthreads();
    if (lane == 0) part_s[warp] = top;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_s[w]);
    const float w = fast_exp2(st.x - (top == kNegInf ? 0.f : top));
    float sum = w * st.y;
    weight_s[tid] = w;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    __syncthreads();
    if (lane == 0) part_s[warp] = sum;
    __syncthreads();
    sum = 0.f;
    for (int i = 0; i < kWarps; ++i) sum += part_s[i];
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = lane * 4; d < D; d += 128) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d < a.head_dim) {
#pragma unroll 4
        for (int p = warp; p < parts; p += kWarps) {
          const float f = weight_s[p];
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + part_row(p, row) * D + d);
          acc.x += f * x.x;
          acc.y += f * x.y;
          acc.z += f * x.z;
          acc.w += f * x.w;
        }
      }
      *reinterpret_cast<float4*>(&red_s[warp][d]) = acc;
    }
    __syncthreads();
    if (tid * 4 < a.head_dim) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = 0; i < kWarps; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(&red_s[i][tid * 4]);
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      store4(row, tid * 4, make_float4(acc.x * inverse, acc.y * inverse, acc.z * inverse, acc.w * inverse));
    }
  }
}

// How a head layout is cut: padded head dim, query heads an item takes (8 or 16), kv heads a CTA takes.
struct Shape {
  int D, nt, heads_cta, row_chunks;
};
Shape shape_of(int head_dim, int heads_q, int heads_kv) {
  Shape s;
  s.D = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  const int group = heads_q / heads_kv;
  s.nt = group > 8 && s.D <= 128 ? 2 : 1;
  s.row_chunks = (group + s.nt * 8 - 1) / (s.nt * 8);
  s.heads_cta = 8;
  while (heads_kv % s.heads_cta) s.heads_cta /= 2;
  return s;
}

int cta_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    cudaGetLastError();
    return set_error(FA_ERR_DEVICE, "cannot query the SM count of the current device");
  }
  return sms < kMaxCtas ? sms : kMaxCtas;
}

int64_t prefix_bytes(int batch) { return ((int64_t)(batch + 1) * 8 + 15) / 16 * 16; }

template <typename C8, int D, int NT>
int launch(const Args& a, int ctas, cudaStream_t stream) {
  auto kernel = paged8_kernel<C8, D, NT>;
  constexpr int smem = Smem<D, NT>::kBytes;
  static_assert(smem <= 227 * 1024 - 256, "shared memory of an SM");
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) {
    kernel<<<ctas, kThreads, smem, stream>>>(a);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && ctas > 1) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas - 1);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, paged8_merge_kernel<D, NT>, a, ctas);
  }
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return set_error(FA_ERR_LAUNCH, "8-bit paged decode launch failed: %s", cudaGetErrorString(e));
}

template <typename C8>
int dispatch(const Shape& s, const Args& a, int ctas, cudaStream_t stream) {
  if (s.D == 64) return s.nt == 1 ? launch<C8, 64, 1>(a, ctas, stream) : launch<C8, 64, 2>(a, ctas, stream);
  if (s.D == 128) return s.nt == 1 ? launch<C8, 128, 1>(a, ctas, stream) : launch<C8, 128, 2>(a, ctas, stream);
  return launch<C8, 256, 1>(a, ctas, stream);
}

}  // namespace

int64_t paged8_workspace_bytes(const fa_paged8_params& p) {
  const int ctas = cta_count();
  if (ctas < 0) return ctas;
  const Shape s = shape_of(p.head_dim, p.heads_q, p.heads_kv);
  return prefix_bytes(p.batch) + (int64_t)2 * ctas * item_rows(s.heads_cta, s.nt) * (s.D + 2) * 4;
}

int launch_decode_paged8(const fa_paged8_params& p, cudaStream_t stream) {
  const int ctas = cta_count();
  if (ctas < 0) return ctas;
  const Shape s = shape_of(p.head_dim, p.heads_q, p.heads_kv);
  for (int i = 0; i < 2; ++i)
    if ((uint64_t)p.k_strides[i] > UINT32_MAX || (uint64_t)p.v_strides[i] > UINT32_MAX)
      return set_error(FA_ERR_UNSUPPORTED, "8-bit paged decode: block and token strides must be below 2^32");
  if (((int64_t)p.max_blocks * p.block_size) > INT32_MAX)
    return set_error(FA_ERR_UNSUPPORTED, "8-bit paged decode: a block table of more than 2^31 - 1 tokens");
  Args a = {};
  a.dtype = p.dtype;
  a.batch = p.batch;
  a.heads_q = p.heads_q;
  a.heads_kv = p.heads_kv;
  a.head_dim = p.head_dim;
  a.group = p.heads_q / p.heads_kv;
  a.num_blocks = p.num_blocks;
  a.max_blocks = p.max_blocks;
  while ((1 << a.shift) < p.block_size) ++a.shift;
  a.head_ctas = p.heads_kv / s.heads_cta;
  a.row_chunks = s.row_chunks;
  a.warps_per_head = kWarps / s.heads_cta;
  a.q = p.q;
  a.q_sb = p.q_strides[0];
  a.q_sh = p.q_strides[1];
  a.k = static_cast<const uint8_t*>(p.k_cache);
  a.v = static_cast<const uint8_t*>(p.v_cache);
  a.k_sb = (uint32_t)p.k_strides[0];
  a.k_st = (uint32_t)p.k_strides[1];
  a.k_sh = p.k_strides[2];
  a.v_sb = (uint32_t)p.v_strides[0];
  a.v_st = (uint32_t)p.v_strides[1];
  a.v_sh = p.v_strides[2];
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
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  a.prefix = reinterpret_cast<int64_t*>(ws);
  a.part_stat = reinterpret_cast<float*>(ws + prefix_bytes(p.batch));
  a.part_o = a.part_stat + (int64_t)2 * ctas * item_rows(s.heads_cta, s.nt) * 2;
  return p.cache_dtype == FA_CACHE_E4M3 ? dispatch<CodeE4M3>(s, a, ctas, stream)
                                        : dispatch<CodeInt8>(s, a, ctas, stream);
}

}  // namespace fa
