// Penalties, bias and grammar mask on the logits of a sampling step.
//
//   x -> x > 0 ? x / r : x r     if the token occurs in the row's history (prompt and generated tokens)
//     -> x - presence [c > 0] - frequency c     c = occurrences among the generated tokens
//     -> x + bias,  -inf where the row's bit mask has a zero
//
// One block per (piece of the vocabulary, row): the piece's occurrence counts are built in shared memory by integer
// atomics (their order does not matter) from the row's history, then the piece is streamed once.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

constexpr int LG_PIECE = 4096;

template <typename T>
__device__ __forceinline__ float lg_load(const T* p) { return static_cast<float>(*p); }
template <typename T>
__device__ __forceinline__ void lg_store(T* p, float x) { *p = static_cast<T>(x); }

template <typename T>
__global__ void __launch_bounds__(256) penalize_kernel(const LbPenalizeArgs a) {
  __shared__ int cnt[LG_PIECE];  // low 31 bits: generated occurrences; sign bit: seen at all
  const int row = blockIdx.y, v0 = blockIdx.x * LG_PIECE, n = min(LG_PIECE, a.V - v0);
  for (int i = threadIdx.x; i < LG_PIECE; i += 256) cnt[i] = 0;
  __syncthreads();
  const int total = max(0, min(a.history_len[row], a.L));
  const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
  for (int i = threadIdx.x; i < total; i += 256) {
    const long long t = a.history[row * a.history_stride + i] - v0;
    if (t >= 0 && t < n) {
      atomicOr(&cnt[t], (int)0x80000000);
      if (i >= prompt) atomicAdd(&cnt[t], 1);
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : a.repetition_s;
  const float pres = a.presence ? a.presence[row] : a.presence_s;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_s;
  const T* in = (const T*)a.logits + row * a.ld_in + v0;
  T* out = (T*)a.out + row * a.ld_out + v0;
  for (int i = threadIdx.x; i < n; i += 256) {
    float x = lg_load(in + i);
    const int c = cnt[i];
    if (c) {
      x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;  // the fast-math division is off by more than a step
      const int g = c & 0x7FFFFFFF;
      if (g) x -= pres + freq * (float)g;
    }
    if (a.bias) x += a.bias[row * a.bias_stride + v0 + i];
    if (a.allowed && !((a.allowed[row * a.allowed_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
    lg_store(out + i, x);
  }
}

}  // namespace lb

extern "C" int lb_penalize_logits(const LbPenalizeArgs* a, void* stream) {
  using namespace lb;
  if (a->dtype != LB_BF16 && a->dtype != LB_F32) return 1;
  if (a->N > 65535) return 2;
  if (a->N <= 0 || a->V <= 0) return 0;
  const dim3 grid((a->V + LG_PIECE - 1) / LG_PIECE, a->N);
  if (a->dtype == LB_BF16)
    penalize_kernel<__nv_bfloat16><<<grid, 256, 0, (cudaStream_t)stream>>>(*a);
  else
    penalize_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>(*a);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}
