// Attention of new tokens over a paged KV cache (see paged_cache.cu for the layout of cache and batch).
//
// The query of a token at position p sees the keys j <= p of its sequence and, with a sliding window W, of those only
// the ones with j > p - W or j < sinks. A row that sees no key (a padding row, an empty sequence) gives zeros.
//
// One block per (token, head): four warps stride over the keys with one online softmax each (running maximum m,
// sum l, accumulator), joined in shared memory at the end.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

template <int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(const LbPagedAttnArgs a) {
  constexpr int E = D / 32;  // channels of a lane
  const int tok = blockIdx.x, h = blockIdx.y, hk = h / (a.H / a.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int seq = tok, n_new = 1, at = 0;
  if (a.cu_q) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
    }
    seq = lo;
    n_new = a.cu_q[seq + 1] - a.cu_q[seq];
    at = tok - a.cu_q[seq];
    if (at < 0 || at >= n_new) seq = -1;
  }
  long long n = 0;  // visible keys end here
  if (seq >= 0) n = (long long)a.kv_len[seq] - n_new + at + 1;
  if (n > (long long)a.cols * a.page) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, ST_BAD_ARG | 0x43u);
    n = (long long)a.cols * a.page;
  }
  float q[E], acc[E], m = -INFINITY, l = 0.f;
  const __nv_bfloat16* qp = (const __nv_bfloat16*)a.q + tok * a.q_st + h * a.q_sh + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) { q[e] = __bfloat162float(qp[e]) * a.scale; acc[e] = 0.f; }
  const long long w0 = a.window > 0 ? n - a.window : 0;
  for (long long j = warp; j < n; j += 4) {
    if (j < w0 && j >= a.sinks) { j += (w0 - j) / 4 * 4; if (j < w0) continue; }
    const int page = a.table[seq * a.table_stride + j / a.page];
    if (page < 0 || page >= a.n_pages) {
      if (lane == 0 && a.status) atomicOr(a.status, ST_BAD_ARG | 0x44u);
      continue;
    }
    const __nv_bfloat16* kp = (const __nv_bfloat16*)a.k_pages + page * a.kp_sp + (j % a.page) * a.kp_st + hk * a.kp_sh + lane * E;
    const __nv_bfloat16* vp = (const __nv_bfloat16*)a.v_pages + page * a.vp_sp + (j % a.page) * a.vp_st + hk * a.vp_sh + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * __bfloat162float(kp[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    const float mn = fmaxf(m, s), corr = __expf(m - mn), p = __expf(s - mn);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * corr + p * __bfloat162float(vp[e]);
    l = l * corr + p;
    m = mn;
  }
  __shared__ float sm_m[4], sm_l[4], sm_acc[4][D];
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < E; ++e) sm_acc[warp][lane * E + e] = acc[e];
  __syncthreads();
  if (threadIdx.x < D) {
    const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float c = sm_m[w] == -INFINITY ? 0.f : __expf(sm_m[w] - M);
      L += sm_l[w] * c;
      o += sm_acc[w][threadIdx.x] * c;
    }
    ((__nv_bfloat16*)a.o)[((long long)tok * a.H + h) * D + threadIdx.x] = __float2bfloat16(L > 0.f ? o / L : 0.f);
  }
}

}  // namespace lb

extern "C" int lb_paged_attention(const LbPagedAttnArgs* a, void* stream) {
  using namespace lb;
  if (a->D != 64 && a->D != 128) return 1;
  if (a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->H > 65535) return 2;
  if (a->T <= 0) return 0;
  const dim3 grid(a->T, a->H);
  if (a->D == 128)
    paged_attn_kernel<128><<<grid, 128, 0, (cudaStream_t)stream>>>(*a);
  else
    paged_attn_kernel<64><<<grid, 128, 0, (cudaStream_t)stream>>>(*a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}
