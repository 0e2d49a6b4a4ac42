// Decode attention over a paged 8-bit cache (fa_decode_paged8).
#include "fa_paged8.cuh"

namespace fa {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;

// One CTA a (request, query head); a warp takes every fourth token with an online softmax of its own.
template <typename C8>
__global__ void __launch_bounds__(kThreads) paged8_kernel(const fa_paged8_params a, int shift) {
  __shared__ float o_s[kWarps][kMaxDim], m_s[kWarps], l_s[kWarps];
  const int b = blockIdx.y, hq = blockIdx.x, head = hq / (a.heads_q / a.heads_kv);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t cap = (int64_t)a.max_blocks << shift;
  const int len = (int)max((int64_t)0, min((int64_t)a.context_lens[b * a.cl_stride], cap));
  float q[kMaxDim / 32], o[kMaxDim / 32], m = kNegInf, l = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxDim / 32; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < a.head_dim ? load_as_float(a.q, b * a.q_strides[0] + hq * a.q_strides[1] + d, a.dtype) : 0.f;
    o[i] = 0.f;
  }
  const uint8_t* kc = static_cast<const uint8_t*>(a.k_cache) + head * a.k_strides[2];
  const uint8_t* vc = static_cast<const uint8_t*>(a.v_cache) + head * a.v_strides[2];
  for (int t = warp; t < len; t += kWarps) {
    const int id = a.block_table[b * a.bt_strides[0] + (t >> shift) * a.bt_strides[1]];
    if (id < 0 || id >= a.num_blocks) continue;
    const int within = t & ((1 << shift) - 1);
    const uint8_t* k = kc + id * a.k_strides[0] + within * a.k_strides[1];
    const uint8_t* v = vc + id * a.v_strides[0] + within * a.v_strides[1];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxDim / 32; ++i) {
      const int d = lane + 32 * i;
      if (d < a.head_dim) dot += q[i] * DType<__half>::unpack2(C8::lo(k[d])).x;
    }
    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
    const float s = dot * a.softmax_scale * a.k_scales[id * a.ks_strides[0] + head * a.ks_strides[1]];
    const float m_new = fmaxf(m, s), alpha = m_new == kNegInf ? 1.f : expf(m - m_new), p = expf(s - m_new);
    const float pv = p * a.v_scales[id * a.vs_strides[0] + head * a.vs_strides[1]];
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < kMaxDim / 32; ++i) {
      const int d = lane + 32 * i;
      if (d < a.head_dim) o[i] = o[i] * alpha + pv * DType<__half>::unpack2(C8::lo(v[d])).x;
    }
  }
#pragma unroll
  for (int i = 0; i < kMaxDim / 32; ++i) o_s[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  float M = kNegInf, L = 0.f, w[kWarps];
  for (int i = 0; i < kWarps; ++i) M = fmaxf(M, m_s[i]);
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    w[i] = M == kNegInf ? 0.f : expf(m_s[i] - M);
    L += w[i] * l_s[i];
  }
  for (int d = threadIdx.x; d < a.head_dim; d += kThreads) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) x += w[i] * o_s[i][d];
    store_from_float(a.out, b * a.o_strides[0] + hq * a.o_strides[1] + d, a.dtype, L == 0.f ? 0.f : x / L);
  }
}

}  // namespace

int64_t paged8_workspace_bytes(const fa_paged8_params&) { return 16; }

int launch_decode_paged8(const fa_paged8_params& p, cudaStream_t stream) {
  if (p.batch > 65535) return set_error(FA_ERR_UNSUPPORTED, "8-bit paged decode takes at most 65535 sequences");
  int shift = 0;
  while ((1 << shift) < p.block_size) ++shift;
  const dim3 grid(p.heads_q, p.batch);
  if (p.cache_dtype == FA_CACHE_E4M3) paged8_kernel<CodeE4M3><<<grid, kThreads, 0, stream>>>(p, shift);
  else paged8_kernel<CodeInt8><<<grid, kThreads, 0, stream>>>(p, shift);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FA_ERR_LAUNCH, "8-bit paged decode launch failed: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace fa
