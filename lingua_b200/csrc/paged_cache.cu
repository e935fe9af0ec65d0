// Writing to and moving pages of a paged KV cache.
//
// A cache layer is two pools [n_pages, page, Hkv, D] (keys, values); row `seq` of the block table names the page of
// every `page` consecutive positions of a sequence. The new tokens of a step are packed rows: token t belongs to the
// sequence with cu_q[seq] <= t < cu_q[seq + 1] (without cu_q: one token per sequence) and the last of them stands at
// position kv_len[seq] - 1.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

// One thread per 16-byte vector (8 channels) of a token; it walks over the heads with stride gridDim.y.
__global__ void __launch_bounds__(256) paged_append_kernel(const LbPagedAppendArgs a) {
  const int vph = a.D / 8;
  const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= (long long)a.T * vph) return;
  const int tok = (int)(i / vph), v = (int)(i % vph);
  int seq = tok, n_new = 1, at = 0;
  if (a.cu_q) {
    // last sequence whose first row is <= tok (empty sequences share their first row with the next one)
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
    }
    seq = lo;
    const int c0 = a.cu_q[seq], c1 = a.cu_q[seq + 1];
    n_new = c1 - c0;
    at = tok - c0;
    if (tok < c0 || tok >= c1) seq = -1;  // a padding row
  }
  long long pos = -1;
  if (seq >= 0) pos = (long long)a.kv_len[seq] - n_new + at;
  __nv_bfloat16 *kd = nullptr, *vd = nullptr;
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (pos >= 0) {
    const long long col = pos / a.page;
    const int page = col < a.cols ? a.table[seq * a.table_stride + col] : -1;
    if (page < 0 || page >= a.n_pages || (a.cs && pos >= a.cs_rows)) {
      if (a.status) atomicOr(a.status, ST_BAD_ARG | 0x41u);
      pos = -1;
    } else {
      const long long row = pos % a.page;
      kd = (__nv_bfloat16*)a.k_pages + page * a.kp_sp + row * a.kp_st + v * 8;
      vd = (__nv_bfloat16*)a.v_pages + page * a.vp_sp + row * a.vp_st + v * 8;
      if (a.cs) {
        const float4* c4 = reinterpret_cast<const float4*>(a.cs + (pos * (a.D / 2) + v * 4) * 2);
        const float4 x = __ldg(c4), y = __ldg(c4 + 1);
        c[0] = x.x; s[0] = x.y; c[1] = x.z; s[1] = x.w;
        c[2] = y.x; s[2] = y.y; c[3] = y.z; s[3] = y.w;
      }
    }
  }
  auto rotate = [&](uint4 u) {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
      w[j] = pack_bf16(f.x * c[j] - f.y * s[j], f.x * s[j] + f.y * c[j]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int h = blockIdx.y; h < a.H + 2 * a.Hkv; h += gridDim.y) {
    if (h < a.H) {
      uint4 u = zero;
      if (pos >= 0) {
        u = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + tok * a.q_st + h * a.q_sh + v * 8);
        if (a.cs) u = rotate(u);
      }
      *reinterpret_cast<uint4*>((__nv_bfloat16*)a.q_out + ((long long)tok * a.H + h) * a.D + v * 8) = u;
    } else if (pos >= 0 && h < a.H + a.Hkv) {
      const int g = h - a.H;
      uint4 u = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.k + tok * a.k_st + g * a.k_sh + v * 8);
      if (a.cs) u = rotate(u);
      *reinterpret_cast<uint4*>(kd + g * a.kp_sh) = u;
    } else if (pos >= 0) {
      const int g = h - a.H - a.Hkv;
      *reinterpret_cast<uint4*>(vd + g * a.vp_sh) =
          *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.v + tok * a.v_st + g * a.v_sh + v * 8);
    }
  }
}

// pool[r, dst[i]] = pool[r, src[i]] for every row r: grid (pieces of a page, rows, pairs)
__global__ void __launch_bounds__(256) copy_pages_kernel(char* pool, long long sr, long long sp, long long bytes,
                                                         int n_pages, const int* src, const int* dst,
                                                         uint32_t* status) {
  const int from = src[blockIdx.z], to = dst[blockIdx.z];
  if (from < 0 || from >= n_pages || to < 0 || to >= n_pages) {
    if (threadIdx.x == 0 && status) atomicOr(status, ST_BAD_ARG | 0x42u);
    return;
  }
  const uint4* s = reinterpret_cast<const uint4*>(pool + blockIdx.y * sr + from * sp);
  uint4* d = reinterpret_cast<uint4*>(pool + blockIdx.y * sr + to * sp);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < bytes / 16; i += gridDim.x * 256ll) d[i] = s[i];
}

}  // namespace lb

extern "C" int lb_paged_append(const LbPagedAppendArgs* a, void* stream) {
  using namespace lb;
  if (a->D != 64 && a->D != 128) return 1;
  if (a->H <= 0 || a->Hkv <= 0 || a->page <= 0) return 2;
  if (a->T <= 0) return 0;
  const long long threads = (long long)a->T * (a->D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), a->H + 2 * a->Hkv);
  paged_append_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(*a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

extern "C" int lb_copy_pages(void* pool, long long row_bytes, long long page_stride_bytes, long long page_bytes,
                             int rows, int n_pages, const int* src, const int* dst, int n, uint32_t* status,
                             void* stream) {
  using namespace lb;
  if (page_bytes % 16 || row_bytes % 16 || page_stride_bytes % 16) return 1;
  if (n > 65535 || rows > 65535) return 2;
  if (n <= 0 || rows <= 0 || page_bytes <= 0) return 0;
  const long long per = (page_bytes / 16 + 255) / 256;
  const dim3 grid((unsigned)(per < 8 ? per : 8), rows, n);
  copy_pages_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>((char*)pool, row_bytes, page_stride_bytes, page_bytes,
                                                            n_pages, src, dst, status);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}
