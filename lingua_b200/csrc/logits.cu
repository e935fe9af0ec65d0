// Penalties, bias and grammar mask on the logits of a sampling step.
//
//   x -> x > 0 ? x / r : x r     if the token occurs in the row's history (prompt and generated tokens)
//     -> x - presence [c > 0] - frequency c     c = occurrences among the generated tokens
//     -> x + bias,  -inf where the row's bit mask has a zero
//
// Bound by the logits' bytes (read and written once). One block per (piece of the vocabulary, row). Every thread first
// issues the loads of its part of the piece and of the history; then the block counts the occurrences of the piece's
// tokens in the history, in shared memory, by integer atomics (their order does not matter). The history is read
// once per piece, from L2. 64 x 128256 fp32 with 2000 entries, bias and mask (68 MB): 16.6 us in a graph, of which 5 us are
// the counting; twice the threads 15.5 us but slower in bf16, half the vectors 17.3 us.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

constexpr int LG_THREADS = 256;
constexpr int LG_VECS = 4;  // 16-byte vectors of a thread
constexpr int LG_HIST = 8;  // history entries of a thread that are requested together with the logits

template <typename T> struct LgVec;
template <> struct LgVec<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct LgVec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
  __device__ static uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
};

template <typename T>
__global__ void __launch_bounds__(LG_THREADS, 4) penalize_kernel(const LbPenalizeArgs a) {
  using Vec = LgVec<T>;
  constexpr int PIECE = LG_THREADS * LG_VECS * Vec::N;
  __shared__ __align__(16) int cnt[PIECE];  // low 31 bits: generated occurrences; sign bit: seen at all
  const int row = blockIdx.y, v0 = blockIdx.x * PIECE, n = min(PIECE, a.V - v0);
  const T* in = (const T*)a.logits + row * a.ld_in + v0;
  T* out = (T*)a.out + row * a.ld_out + v0;
  const float* bias = a.bias ? a.bias + row * a.bias_stride + v0 : nullptr;
  // whole vectors where the row's addresses allow them, single elements at the end of the row or of an odd row
  const bool even = (((uintptr_t)in | (uintptr_t)out | (uintptr_t)bias) & 15) == 0;
  const int n_vec = even ? n / Vec::N : 0;
  uint4 x[LG_VECS];
#pragma unroll
  for (int u = 0; u < LG_VECS; ++u) {
    const int i = u * LG_THREADS + threadIdx.x;
    if (i < n_vec) x[u] = reinterpret_cast<const uint4*>(in)[i];
  }
  const long long* hist = a.history + row * a.history_stride;
  long long id[LG_HIST];
#pragma unroll
  for (int u = 0; u < LG_HIST; ++u) {
    const int i = u * LG_THREADS + threadIdx.x;
    if (i < a.L) id[u] = __ldg(hist + i);
  }
  for (int i = threadIdx.x; i < (n + 3) / 4; i += LG_THREADS) reinterpret_cast<int4*>(cnt)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  const int total = max(0, min(a.history_len[row], a.L));
  const int prompt = a.prompt_len ? a.prompt_len[row] : 0;
  auto count = [&](int i, long long token) {
    const long long t = token - v0;
    if (t >= 0 && t < n) {
      atomicOr(&cnt[t], (int)0x80000000);
      if (i >= prompt) atomicAdd(&cnt[t], 1);
    }
  };
#pragma unroll
  for (int u = 0; u < LG_HIST; ++u) {
    const int i = u * LG_THREADS + threadIdx.x;
    if (i < total) count(i, id[u]);
  }
  for (int i = LG_HIST * LG_THREADS + threadIdx.x; i < total; i += LG_THREADS) count(i, hist[i]);
  const float rep = a.repetition ? a.repetition[row] : a.repetition_s;
  const float pres = a.presence ? a.presence[row] : a.presence_s;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_s;
  const uint32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride + (v0 >> 5) : nullptr;
  __syncthreads();
  auto one = [&](float z, int c, float b, bool ok) {
    if (c) {
      z = z > 0.f ? __fdiv_rn(z, rep) : z * rep;  // the fast-math division is off by more than a step
      const int g = c & 0x7FFFFFFF;
      if (g) z -= pres + freq * (float)g;
    }
    return ok ? z + b : -INFINITY;
  };
#pragma unroll
  for (int u = 0; u < LG_VECS; ++u) {
    const int i = u * LG_THREADS + threadIdx.x;
    if (i < n_vec) {
      float f[Vec::N];
      Vec::unpack(x[u], f);
      const uint32_t ok = allowed ? allowed[(i * Vec::N) >> 5] >> ((i * Vec::N) & 31) : 0xFFFFFFFFu;
#pragma unroll
      for (int e = 0; e < Vec::N; e += 4) {
        const int4 c = *reinterpret_cast<const int4*>(cnt + i * Vec::N + e);
        const float4 b = bias ? __ldg(reinterpret_cast<const float4*>(bias + i * Vec::N + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
        f[e] = one(f[e], c.x, b.x, ok >> e & 1);
        f[e + 1] = one(f[e + 1], c.y, b.y, ok >> (e + 1) & 1);
        f[e + 2] = one(f[e + 2], c.z, b.z, ok >> (e + 2) & 1);
        f[e + 3] = one(f[e + 3], c.w, b.w, ok >> (e + 3) & 1);
      }
      reinterpret_cast<uint4*>(out)[i] = Vec::pack(f);
    }
  }
#pragma unroll 4
  for (int i = n_vec * Vec::N + threadIdx.x; i < n; i += LG_THREADS)
    out[i] = static_cast<T>(one(static_cast<float>(in[i]), cnt[i], bias ? bias[i] : 0.f,
                                !allowed || (allowed[i >> 5] >> (i & 31) & 1)));
}

template <typename T>
static void launch_penalize(const LbPenalizeArgs& a, cudaStream_t st) {
  constexpr int PIECE = LG_THREADS * LG_VECS * LgVec<T>::N;
  penalize_kernel<T><<<dim3((a.V + PIECE - 1) / PIECE, a.N), LG_THREADS, 0, st>>>(a);
}

}  // namespace lb

extern "C" int lb_penalize_logits(const LbPenalizeArgs* a, void* stream) {
  using namespace lb;
  if (a->dtype != LB_BF16 && a->dtype != LB_F32) return 1;
  if (a->N > 65535) return 2;
  if (a->N <= 0 || a->V <= 0) return 0;
  if (a->dtype == LB_BF16)
    launch_penalize<__nv_bfloat16>(*a, (cudaStream_t)stream);
  else
    launch_penalize<float>(*a, (cudaStream_t)stream);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}
