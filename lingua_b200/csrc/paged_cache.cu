// Writing to and moving pages of a paged KV cache.
//
// A cache layer is two pools [n_pages, page, Hkv, D] (keys, values); row `seq` of the block table names the page of
// every `page` consecutive positions of a sequence. The new tokens of a step are packed rows: token t belongs to the
// sequence with cu_q[seq] <= t < cu_q[seq + 1] (without cu_q: one token per sequence) and the last of them stands at
// position kv_len[seq] - 1.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

// Bound by its bytes: every row is read and written once, 16 bytes at a time. A thread owns one 16-byte vector position
// (8 channels, 4 rotation pairs) of a token and AP_HEADS of its heads, so that position, page and cos / sin row are found
// once for all of them; the heads' loads are issued before that search (sequence, length, page: a chain of dependent reads)
// and arrive while it runs. 24 prompts, 2532 tokens of 48
// heads (64 MB): 10.7 us, 6.0 TB/s, in a graph (one head to a thread: 31 us a call, now 17 us, most of it the host's).
constexpr int AP_HEADS = 8;
__global__ void __launch_bounds__(128) paged_append_kernel(const LbPagedAppendArgs a) {
  const int vph = a.D / 8, v = threadIdx.x & (vph - 1);  // 8 or 16 vectors of a head
  const int tok = blockIdx.x * (128 / vph) + threadIdx.x / vph;
  if (tok >= a.T) return;
  const int h0 = blockIdx.y * AP_HEADS, n_heads = min(AP_HEADS, a.H + 2 * a.Hkv - h0);
  uint4 x[AP_HEADS];
#pragma unroll
  for (int u = 0; u < AP_HEADS; ++u) {
    const int h = h0 + u;
    if (u < n_heads) {
      const __nv_bfloat16* p = h < a.H ? (const __nv_bfloat16*)a.q + tok * a.q_st + h * a.q_sh
                               : h < a.H + a.Hkv ? (const __nv_bfloat16*)a.k + tok * a.k_st + (h - a.H) * a.k_sh
                                                 : (const __nv_bfloat16*)a.v + tok * a.v_st + (h - a.H - a.Hkv) * a.v_sh;
      x[u] = __ldg(reinterpret_cast<const uint4*>(p + v * 8));
    }
  }
  int seq = tok, n_new = 1, at = 0;
  if (a.cu_q) {
    // last sequence whose first row is <= tok (empty sequences share their first row with the next one)
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
    }
    seq = lo;
    const int c0 = a.n_seqs > 0 ? a.cu_q[seq] : 0, c1 = a.n_seqs > 0 ? a.cu_q[seq + 1] : 0;
    n_new = c1 - c0;
    at = tok - c0;
    if (tok < c0 || tok >= c1) seq = -1;  // a padding row
  }
  const int page_log = __ffs(a.page) - 1;
  long long pos = -1;
  if (seq >= 0) pos = (long long)a.kv_len[seq] - n_new + at;
  __nv_bfloat16 *kd = nullptr, *vd = nullptr;
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (pos >= 0) {
    const int col = (int)min(pos >> page_log, 0x7FFFFFFFll);
    const int page = col < a.cols ? a.table[seq * a.table_stride + col] : -1;
    if (page < 0 || page >= a.n_pages || (a.cs && pos >= a.cs_rows)) {
      if (a.status) atomicOr(a.status, ST_BAD_ARG | 0x41u);
      pos = -1;
    } else {
      const int row = (int)pos & (a.page - 1);
      kd = (__nv_bfloat16*)a.k_pages + page * a.kp_sp + row * a.kp_st + v * 8;
      vd = (__nv_bfloat16*)a.v_pages + page * a.vp_sp + row * a.vp_st + v * 8;
      if (a.cs) {
        const float4* c4 = reinterpret_cast<const float4*>(a.cs + (pos * (a.D / 2) + v * 4) * 2);
        const float4 y = __ldg(c4), z = __ldg(c4 + 1);
        c[0] = y.x; s[0] = y.y; c[1] = y.z; s[1] = y.w;
        c[2] = z.x; s[2] = z.y; c[3] = z.z; s[3] = z.w;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < AP_HEADS; ++u) {
    const int h = h0 + u;
    if (u >= n_heads) break;
    if (a.cs && h < a.H + a.Hkv) {
      uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
        w[j] = pack_bf16(f.x * c[j] - f.y * s[j], f.x * s[j] + f.y * c[j]);
      }
      x[u] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (h < a.H) {
      *reinterpret_cast<uint4*>((__nv_bfloat16*)a.q_out + ((long long)tok * a.H + h) * a.D + v * 8) =
          pos >= 0 ? x[u] : make_uint4(0, 0, 0, 0);
    } else if (pos >= 0) {
      *reinterpret_cast<uint4*>(h < a.H + a.Hkv ? kd + (h - a.H) * a.kp_sh : vd + (h - a.H - a.Hkv) * a.vp_sh) = x[u];
    }
  }
}

// pool[r, dst[i]] = pool[r, src[i]] for every row r. The 16-byte vectors of a page, all rows one after the other, are one
// list; a block moves 2048 of them (32 KB), each thread eight with all loads in flight before the first store. Bound by DRAM:
// 61 pages of 50 x 262 KB in 243 us, 6.6 TB/s (one vector in flight per thread: 258 us); 64 of 50 x 64 KB in 68 us (78 us).
constexpr int CP_VECS = 8;
__global__ void __launch_bounds__(256) copy_pages_kernel(char* pool, long long sr, long long sp, uint32_t vecs,
                                                         long long total, int n_pages, const int* src, const int* dst,
                                                         uint32_t* status) {
  const int from = src[blockIdx.y], to = dst[blockIdx.y];
  if (from < 0 || from >= n_pages || to < 0 || to >= n_pages) {
    if (threadIdx.x == 0 && status) atomicOr(status, ST_BAD_ARG | 0x42u);
    return;
  }
  const long long gap = (to - from) * sp;
  uint4 x[CP_VECS];
  char* p[CP_VECS];
#pragma unroll
  for (int u = 0; u < CP_VECS; ++u) {
    const long long i = blockIdx.x * (256ll * CP_VECS) + u * 256 + threadIdx.x;
    p[u] = nullptr;
    if (i < total) {
      // position in the list -> row and vector of the page (32-bit division where the list is short enough)
      const long long r = total >> 32 ? i / vecs : (long long)((uint32_t)i / vecs);
      p[u] = pool + r * sr + from * sp + (i - r * vecs) * 16;
      x[u] = *reinterpret_cast<const uint4*>(p[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < CP_VECS; ++u)
    if (p[u]) *reinterpret_cast<uint4*>(p[u] + gap) = x[u];
}

}  // namespace lb

extern "C" int lb_paged_append(const LbPagedAppendArgs* a, void* stream) {
  using namespace lb;
  if (a->D != 64 && a->D != 128) return 1;
  if (a->H <= 0 || a->Hkv <= 0 || a->page <= 0 || (a->page & (a->page - 1))) return 2;
  if (a->T <= 0) return 0;
  const int toks = 128 / (a->D / 8);
  const dim3 grid((a->T + toks - 1) / toks, (a->H + 2 * a->Hkv + AP_HEADS - 1) / AP_HEADS);
  paged_append_kernel<<<grid, 128, 0, (cudaStream_t)stream>>>(*a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

extern "C" int lb_copy_pages(void* pool, long long row_bytes, long long page_stride_bytes, long long page_bytes,
                             int rows, int n_pages, const int* src, const int* dst, int n, uint32_t* status,
                             void* stream) {
  using namespace lb;
  if (page_bytes % 16 || row_bytes % 16 || page_stride_bytes % 16) return 1;
  if (page_bytes / 16 > 0xFFFFFFFFll) return 2;
  if (n <= 0 || rows <= 0 || page_bytes <= 0) return 0;
  const long long vecs = page_bytes / 16, total = vecs * rows, per = 256ll * CP_VECS;
  for (int i = 0; i < n; i += 65535) {  // what a grid dimension holds
    const dim3 grid((unsigned)((total + per - 1) / per), n - i < 65535 ? n - i : 65535);
    copy_pages_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>((char*)pool, row_bytes, page_stride_bytes, (uint32_t)vecs,
                                                              total, n_pages, src + i, dst + i, status);
  }
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}
