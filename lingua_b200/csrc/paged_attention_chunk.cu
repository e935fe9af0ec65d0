// Attention of chunks of new tokens over a paged KV cache on tcgen05 (visibility rule and batch layout: paged_attention.cu).
//
// Bound by the tensor cores: per key tile of 128 and query tile of 128 rows two products of 128 x 128 x D, against
// 2 x 128 x D x 2 bytes of keys and values that 256 rows share. Measured (32 / 8 heads, 128 channels): 2048 tokens over 32768
// keys 864 us, 1230 TFLOP/s (1.05 ms back to back, at the power cap); four prompts of 2048 tokens 162 us. A step takes about
// 3050 cycles where its products alone take 2051: one tile's softmax is longer than the other tile's products. Design:
//  * The rows of a query tile are (token, query head of one kv head) pairs: 128 / G tokens x G heads, loaded by one TMA
//    box. A key tile is thus fetched once for all heads of the group, and short chunks of grouped heads still fill tiles.
//  * An item is (sequence, kv head, pair of query tiles). Its units, CK_ITEM_COST for the item itself and one for each
//    visible key tile of 128, are dealt out, all items in order, in equal contiguous shares to one block per SM. A share that
//    begins or ends inside an item leaves a partial result (row maximum, row sum, unnormalised output in fp32) for the join
//    kernel at the end. So one long chunk of few heads, a batch of odd chunks and a whole prompt all keep 148 SMs equally
//    busy.
//  * Each query tile of the pair has its own softmax warpgroup (a thread owns a whole row of 128 scores, no exchange between
//    threads) and its own S and O in tensor memory. The products of the two tiles alternate,
//        O0 += P0 V(j) | S0 = Q0 K(j+1)^T | O1 += P1 V(j) | S1 = Q1 K(j+1)^T
//    so that one tile's softmax runs under the other tile's products. P goes back to tensor memory over the first half of
//    its S. O is rescaled only when a row maximum grew by more than 2^8.
//  * K and V stages are given back separately (K as soon as both S products of a tile are done), so a K tile is requested
//    about two steps before it is needed. The next item's Q loads under the last step of the previous one.
//  * Keys past the end of a sequence and behind the window lie in the same pages as visible ones. Their scores are
//    replaced by -inf, and their V rows are zeroed in shared memory by the softmax threads before P is handed over (0 x NaN
//    would reach every row). Pages that are missing are requested outside the pool, which TMA fills with zeros.
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

// Control warpgroup (a TMA warp, an MMA warp, two idle ones) and two softmax warpgroups. A softmax thread holds 128
// scores: registers move from the control warps to it, within what the block was launched with (384 x 168 =
// 128 x 104 + 256 x 200).
constexpr int CK_THREADS = 384;
constexpr int CK_REGS_CONTROL = 104, CK_REGS_SOFTMAX = 200;
constexpr int CK_ITEM_COST = 3;     // what beginning and ending an item costs, in key tiles (about 5 us against 1.9 us)
constexpr int CK_HALF = 128 * 128;  // 128 rows x 64 channels: one swizzled box of a tile
constexpr float CK_LOG2E = 1.4426950408889634f;

template <int D>
struct CkCfg {
  static constexpr int NH = D / 64;           // 64-channel halves of a row
  static constexpr int TILE = NH * CK_HALF;   // 128 rows x D
  static constexpr int NST = D == 128 ? 2 : 4;
  static constexpr int SMEM = 2 * TILE + 2 * NST * TILE + 8 * 4096 /* output staging of a softmax warp */ + 1024;
  static constexpr int SLOT = 256 * D + 512;  // floats of a partial result: O, row maxima, row sums
};

struct CkSeq {
  int q0, nq, pos0, end;  // first row of q, new tokens, position of the first one, end of the readable keys
};
struct CkItem {
  int tok0, n_tok0, n_tok1;  // first token, tokens in the two tiles
  int hi0, hi1, lo0, lo1;    // keys [lo, hi) of each tile (and the first tokens)
  int hi, lo;                // of the pair
  int sb, wb, nt;            // key tiles [0, sb), then from wb on; their number
};

__device__ __forceinline__ CkSeq ck_seq(const LbPagedAttnArgs& a, int s, bool report) {
  CkSeq r;
  r.q0 = a.cu_q ? a.cu_q[s] : s;
  r.nq = a.cu_q ? a.cu_q[s + 1] - r.q0 : 1;
  const int cap = a.cols * a.page, len = a.kv_len[s];
  if (report && len > cap && a.status) atomicOr(a.status, ST_BAD_ARG | 0x53u);
  if (r.q0 < 0 || r.nq < 0 || r.q0 > a.T - r.nq) {
    if (report && a.status) atomicOr(a.status, ST_BAD_ARG | 0x55u);
    r.nq = 0;
  }
  r.pos0 = max(len, 0) - r.nq;
  r.end = max(0, min(len, cap));
  return r;
}

__device__ __forceinline__ CkItem ck_item(const LbPagedAttnArgs& a, const CkSeq& q, int pair, int tpt) {
  CkItem t;
  t.tok0 = pair * 2 * tpt;
  t.n_tok0 = max(0, min(tpt, q.nq - t.tok0));
  t.n_tok1 = max(0, min(tpt, q.nq - t.tok0 - tpt));
  const int p0 = q.pos0 + t.tok0, p1 = p0 + tpt;
  t.hi0 = max(0, min(q.end, p0 + t.n_tok0));
  t.hi1 = t.n_tok1 > 0 ? max(0, min(q.end, p1 + t.n_tok1)) : 0;
  t.hi = max(t.hi0, t.hi1);
  t.lo0 = a.window > 0 ? max(0, min(t.hi, p0 - a.window + 1)) : 0;
  t.lo1 = a.window > 0 ? max(0, min(t.hi, p1 - a.window + 1)) : 0;
  t.lo = t.lo0;
  t.wb = t.lo / 128;
  t.sb = min((min(a.sinks, t.lo) + 127) / 128, t.wb);
  t.nt = max(1, t.sb + (t.hi + 127) / 128 - t.wb);
  return t;
}
__device__ __forceinline__ int ck_tile(const CkItem& t, int i) { return i < t.sb ? i : i - t.sb + t.wb; }
// does query tile `w` of the pair see any key of key tile kt?
__device__ __forceinline__ bool ck_active(const LbPagedAttnArgs& a, const CkItem& t, int w, int kt) {
  const int hi = w ? t.hi1 : t.hi0, lo = w ? t.lo1 : t.lo0;
  return (w ? t.n_tok1 : t.n_tok0) > 0 && kt * 128 < hi && (kt * 128 + 128 > lo || kt * 128 < a.sinks);
}

// A block's place in the list of items; every role of the block walks it the same way.
struct CkWalk {
  int seq, hk, pair, first;  // item and the first of its units that is this block's
  long long left;            // units still to do
};

// Descriptors of the k-th 16-deep slice of a tile: the start address (in units of 16 bytes, the low field) moves by
// 32 bytes inside a 64-channel half of a K-major tile, by 16 rows of 128 bytes of an MN-major one.
__device__ __forceinline__ uint64_t ck_slice_k(uint64_t tile, int k) { return tile + (((k >> 2) * CK_HALF + (k & 3) * 32) >> 4); }
__device__ __forceinline__ uint64_t ck_slice_mn(uint64_t tile, int k) { return tile + (k * 2048 >> 4); }

template <int D>
__global__ void __launch_bounds__(CK_THREADS, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, const LbPagedAttnArgs a, float* ws, int4* hdr) {
  using Cfg = CkCfg<D>;
  constexpr int NST = Cfg::NST, NH = Cfg::NH;
  constexpr uint32_t IDESC_S = make_idesc(128, 128, 1, 1, 0, 0), IDESC_O = make_idesc(128, D, 1, 1, 0, 1);
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag;
  __shared__ uint32_t tmem_slot;
  __shared__ long long warp_sum[CK_THREADS / 32];
  __shared__ CkWalk start;
  __shared__ __align__(8) uint64_t bar_mem[2 + 4 * NST + 8];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto sQ = [&](int t) { return sbase + t * Cfg::TILE; };
  auto sK = [&](int s) { return sbase + (2 + 2 * s) * Cfg::TILE; };
  auto sV = [&](int s) { return sbase + (3 + 2 * s) * Cfg::TILE; };
  const uint32_t bars = smem_u32(bar_mem);
  const uint32_t q_full = bars, q_empty = bars + 8;
  auto k_full = [&](int s) { return bars + 16 + 32 * s; };
  auto v_full = [&](int s) { return bars + 24 + 32 * s; };
  auto k_empty = [&](int s) { return bars + 32 + 32 * s; };
  auto v_empty = [&](int s) { return bars + 40 + 32 * s; };
  auto s_full = [&](int t) { return bars + 16 + 32 * NST + 32 * t; };
  auto p_half = [&](int t) { return bars + 24 + 32 * NST + 32 * t; };
  auto p_full = [&](int t) { return bars + 32 + 32 * NST + 32 * t; };
  auto o_done = [&](int t) { return bars + 40 + 32 * NST + 32 * t; };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.Hkv, tpt = 128 / G;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < NST; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_half(t), 4);
      mbar_init(p_full(t), 4);
      mbar_init(o_done(t), 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  if (tpt * G < 128) {  // rows of the Q tiles that no box covers: zeros instead of whatever was there
    for (int i = threadIdx.x; i < 2 * Cfg::TILE / 16; i += CK_THREADS)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sbase + i * 16), "r"(0) : "memory");
    fence_proxy_async_smem();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this block's share. A warp sums the key tiles of a contiguous run of sequences, its lanes share the pairs.
  const int per = (a.n_seqs + CK_THREADS / 32 - 1) / (CK_THREADS / 32);
  const int s_lo = min(a.n_seqs, warp * per), s_hi = min(a.n_seqs, s_lo + per);
  auto seq_tiles = [&](const CkSeq& q) {  // of one kv head; the same in all lanes
    const int n_pairs = (q.nq + 2 * tpt - 1) / (2 * tpt);
    long long n = 0;
    for (int p = lane; p < n_pairs; p += 32) n += ck_item(a, q, p, tpt).nt + CK_ITEM_COST;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    return n;
  };
  auto bcast = [&](const CkSeq& q, int from) {
    CkSeq r;
    r.q0 = __shfl_sync(0xFFFFFFFFu, q.q0, from);
    r.nq = __shfl_sync(0xFFFFFFFFu, q.nq, from);
    r.pos0 = __shfl_sync(0xFFFFFFFFu, q.pos0, from);
    r.end = __shfl_sync(0xFFFFFFFFu, q.end, from);
    return r;
  };
  long long mine = 0;
  for (int base = s_lo; base < s_hi; base += 32) {
    CkSeq ql = {0, 0, 0, 0};
    if (base + lane < s_hi) ql = ck_seq(a, base + lane, blockIdx.x == 0);
    const int n = min(32, s_hi - base);
    for (int i = 0; i < n; ++i) mine += a.Hkv * seq_tiles(bcast(ql, i));
  }
  if (lane == 0) warp_sum[warp] = mine;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < CK_THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const long long n_blocks = max(1ll, min((long long)gridDim.x, total));  // no share is empty
  const bool busy = blockIdx.x < n_blocks;
  auto share = [&](long long i) { return div_nonneg(total * i, n_blocks); };  // first unit of share i
  const long long u0 = busy ? share(blockIdx.x) : 0, u1 = busy ? share(blockIdx.x + 1) : 0;
  if (u0 < u1 && u0 >= before && u0 < before + mine) {
    long long at = before;
    bool found = false;
    for (int base = s_lo; base < s_hi && !found; base += 32) {
      CkSeq ql = {0, 0, 0, 0};
      if (base + lane < s_hi) ql = ck_seq(a, base + lane, false);
      const int n = min(32, s_hi - base);
      for (int i = 0; i < n && !found; ++i) {
        const CkSeq q = bcast(ql, i);
        const long long one = seq_tiles(q);
        if (u0 < at + a.Hkv * one) {
          found = true;
          const int hk = (int)div_nonneg(u0 - at, one);
          long long rest = u0 - at - hk * one;  // units of this head before u0
          const int n_pairs = (q.nq + 2 * tpt - 1) / (2 * tpt);
          for (int p0 = 0; p0 < n_pairs; p0 += 32) {
            const int nt = p0 + lane < n_pairs ? ck_item(a, q, p0 + lane, tpt).nt + CK_ITEM_COST : 0;
            long long incl = nt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
              if (lane >= o) incl += v;
            }
            const long long all = __shfl_sync(0xFFFFFFFFu, incl, 31);
            if (rest < all) {
              if (rest >= incl - nt && rest < incl) {
                start.seq = base + i; start.hk = hk; start.pair = p0 + lane;
                start.first = (int)(rest - (incl - nt)); start.left = u1 - u0;
              }
              break;
            }
            rest -= all;
          }
        }
        at += a.Hkv * one;
      }
    }
  }
  // rows of q that belong to no sequence
  if (a.cu_q) {
    const int lo = a.n_seqs > 0 ? max(0, min(a.T, a.cu_q[0])) : 0;
    const int hi = a.n_seqs > 0 ? max(lo, min(a.T, a.cu_q[a.n_seqs])) : 0;
    const long long vec = (long long)a.H * D / 8;
    for (int t = blockIdx.x; t < lo + a.T - hi; t += gridDim.x) {
      uint4* row = reinterpret_cast<uint4*>((__nv_bfloat16*)a.o + (long long)(t < lo ? t : hi + t - lo) * a.H * D);
      for (long long i = threadIdx.x; i < vec; i += CK_THREADS) row[i] = make_uint4(0, 0, 0, 0);
    }
  }
  if (threadIdx.x == 0) hdr[blockIdx.x] = make_int4(0, 0, 0, 0);
  __syncthreads();

  auto tS = [&](int t) { return tmem + t * 128; };
  auto tO = [&](int t) { return tmem + 256 + t * 128; };
  // walk over this block's pieces: calls body(sequence, item, kv head, first key tile, one past the last)
  auto walk = [&](auto&& body) {
    if (u0 >= u1) return;
    CkWalk w = start;
    CkSeq q = ck_seq(a, w.seq, false);
    while (w.left > 0) {
      const int n_pairs = (q.nq + 2 * tpt - 1) / (2 * tpt);
      if (w.pair >= n_pairs) {
        w.pair = 0;
        if (n_pairs == 0 || ++w.hk >= a.Hkv) {
          w.hk = 0;
          if (++w.seq >= a.n_seqs) return;
          q = ck_seq(a, w.seq, false);
        }
        continue;
      }
      const CkItem t = ck_item(a, q, w.pair, tpt);
      const int f1 = (int)min((long long)(t.nt + CK_ITEM_COST), w.first + w.left);
      const int i0 = max(0, w.first - CK_ITEM_COST), i1 = max(0, f1 - CK_ITEM_COST);
      if (i1 > i0 && !body(q, t, w, i0, i1)) return;
      w.left -= f1 - w.first;
      w.first = 0;
      ++w.pair;
    }
  };

  // a wait of a whole warp has one outcome for all its lanes
  auto wait_all = [&](uint32_t bar, uint32_t parity, uint32_t site) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, &abort_flag, a.status, site)) != 0;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CK_REGS_CONTROL));
    if (warp == 0) {
      // ---------------------------------------------------------------- TMA
      uint32_t kv = 0, piece = 0;  // key tiles and pieces requested so far
      const int page_log = __ffs(a.page) - 1;
      const int rows = min(a.page, 128);  // rows of a box
      const int n_box = 128 / rows;       // boxes of a key tile
      const uint32_t q_bytes = NH * tpt * G * 128;
      walk([&](const CkSeq& q, const CkItem& t, const CkWalk& w, int i0, int i1) {
        const int* trow = a.table + (long long)w.seq * a.table_stride;
        auto page_of = [&](int i) {  // page of box `lane` of the i-th key tile
          const int key = ck_tile(t, i) * 128 + lane * rows;
          int pg = a.n_pages;
          if (lane < n_box && i < i1 && key < t.hi && (key + rows > t.lo || key < a.sinks)) {
            pg = __ldg(trow + (key >> page_log));
            if (pg < 0 || pg >= a.n_pages) {
              if (a.status) atomicOr(a.status, ST_BAD_ARG | 0x54u);
              pg = a.n_pages;
            }
          }
          return pg;
        };
        int pg = page_of(i0);
        for (int i = i0; i < i1; ++i, ++kv) {
          const int s = kv % NST;
          const uint32_t ph = ((kv / NST) & 1) ^ 1;
          const int off = (ck_tile(t, i) * 128 + lane * rows) & (a.page - 1);
          const int next = page_of(i + 1);
          if (!wait_all(k_empty(s), ph, 0x62)) return false;
          if (lane == 0) mbar_arrive_expect_tx(k_full(s), Cfg::TILE);
          __syncwarp();
          if (lane < n_box)
            for (int h = 0; h < NH; ++h)
              tma_load_4d(sK(s) + h * CK_HALF + lane * rows * 128, &tk, k_full(s), 64 * h, off, w.hk, pg);
          if (!wait_all(v_empty(s), ph, 0x63)) return false;
          if (lane == 0) mbar_arrive_expect_tx(v_full(s), Cfg::TILE);
          __syncwarp();
          if (lane < n_box)
            for (int h = 0; h < NH; ++h)
              tma_load_4d(sV(s) + h * CK_HALF + lane * rows * 128, &tv, v_full(s), 64 * h, off, w.hk, pg);
          pg = next;
          if (i == i0) {  // after the first keys, whose stages come free earlier than the Q tiles
            if (!wait_all(q_empty, (piece & 1) ^ 1, 0x61)) return false;
            if (lane == 0) {
              mbar_arrive_expect_tx(q_full, (t.n_tok1 > 0 ? 2 : 1) * q_bytes);
              for (int s = 0; s < (t.n_tok1 > 0 ? 2 : 1); ++s)
                for (int h = 0; h < NH; ++h)
                  tma_load_4d(sQ(s) + h * CK_HALF, &tq, q_full, 64 * h, w.hk * G, q.q0 + t.tok0 + s * tpt, 0);
            }
            ++piece;
          }
        }
        return true;
      });
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA
      if (elect_one()) {
        uint32_t kv = 0, piece = 0, n_p0 = 0, n_p1 = 0;
        walk([&](const CkSeq& q, const CkItem& t, const CkWalk& w, int i0, int i1) {
          int last0 = -1, last1 = -1;  // last active key tile of each query tile
          for (int i = i1 - 1; i >= i0 && last0 < 0; --i)
            if (ck_active(a, t, 0, ck_tile(t, i))) last0 = i;
          for (int i = i1 - 1; i >= i0 && last1 < 0 && t.n_tok1 > 0; --i)
            if (ck_active(a, t, 1, ck_tile(t, i))) last1 = i;
          bool begun0 = false, begun1 = false;
          // MMAs of one thread run in issue order: S_t(i + 1) overwrites P_t(i) only after O_t += P_t V(i) has read it, and
          // a commit after S_t(i + 1) also covers that product.
          auto issue_s = [&](int s, int st) {
            const uint64_t dq = make_smem_desc(sQ(s), 16, 1024), dk = make_smem_desc(sK(st), 16, 1024);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) umma_f16(tS(s), ck_slice_k(dq, k), ck_slice_k(dk, k), IDESC_S, k != 0);
            umma_commit(s_full(s));
          };
          auto issue_pv = [&](int s, int st, uint32_t& n_p, bool& begun, bool last) -> bool {
            // the first 64 keys' P is multiplied while the softmax warps are still at the other 64
            const uint64_t dv = make_smem_desc(sV(st), CK_HALF, 1024);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              if (!mbar_wait(hf ? p_full(s) : p_half(s), n_p & 1, &abort_flag, a.status, 0x64)) return false;
              tc_fence_after();
#pragma unroll
              for (int k = 4 * hf; k < 4 * hf + 4; ++k)
                umma_f16_ts(tO(s), tS(s) + k * 8, ck_slice_mn(dv, k), IDESC_O, (begun || k != 0) ? 1u : 0u);
            }
            begun = true;
            ++n_p;
            if (last) umma_commit(o_done(s));
            return true;
          };
          auto scores = [&](int i, int s, bool& ready) -> bool {  // S of query tile s for key tile i
            const uint32_t n = kv + (i - i0);
            const int st = n % NST;
            if (!ready) {
              if (!mbar_wait(k_full(st), (n / NST) & 1, &abort_flag, a.status, 0x65)) return false;
              tc_fence_after();
              ready = true;
            }
            if (ck_active(a, t, s, ck_tile(t, i))) issue_s(s, st);
            if (s == 1) umma_commit(k_empty(st));
            if (s == 1 && i + 1 == i1) umma_commit(q_empty);
            return true;
          };
          if (!mbar_wait(q_full, piece & 1, &abort_flag, a.status, 0x66)) return false;
          ++piece;
          tc_fence_after();
          bool ready = false;
          if (!scores(i0, 0, ready) || !scores(i0, 1, ready)) return false;
          for (int i = i0; i < i1; ++i) {
            const uint32_t n = kv + (i - i0);
            const int st = n % NST, kt = ck_tile(t, i);
            const bool a0 = ck_active(a, t, 0, kt), a1 = ck_active(a, t, 1, kt);
            ready = false;
            if (!mbar_wait(v_full(st), (n / NST) & 1, &abort_flag, a.status, 0x67)) return false;
            tc_fence_after();
            if (a0 && !issue_pv(0, st, n_p0, begun0, i == last0)) return false;
            if (i + 1 < i1 && !scores(i + 1, 0, ready)) return false;
            if (a1 && !issue_pv(1, st, n_p1, begun1, i == last1)) return false;
            umma_commit(v_empty(st));
            if (i + 1 < i1 && !scores(i + 1, 1, ready)) return false;
          }
          kv += i1 - i0;
          return true;
        });
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CK_REGS_SOFTMAX));
    const int wt = (warp - 4) >> 2;  // query tile
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tSt = tS(wt) + lane_off, tOt = tO(wt) + lane_off;
    const uint32_t stage = sbase + (2 + 2 * NST) * Cfg::TILE + (warp - 4) * 4096;
    const float sl2 = fmaxf(a.scale * CK_LOG2E, 1e-30f);  // a scale of 0 must not turn -inf into NaN
    const int rt = r / G, rg = r % G;  // token and head of this row
    uint32_t kv = 0, n_s = 0, n_o = 0;
    walk([&](const CkSeq& q, const CkItem& t, const CkWalk& w, int i0, int i1) {
      const int n_tok = wt ? t.n_tok1 : t.n_tok0;
      const int p_first = q.pos0 + t.tok0 + wt * tpt;
      const bool live = rt < n_tok && r < tpt * G;
      const int pos = p_first + rt;
      const int hi = live ? max(0, min(pos + 1, q.end)) : 0;  // this row sees keys below hi ...
      const int lo = a.window > 0 ? pos - a.window + 1 : 0;   // ... from lo on, and the first `sinks`
      // key tiles inside [full_lo, full_hi) (or the first tokens) are seen by every row
      const int full_hi = min(p_first + 1, q.end), full_lo = a.window > 0 ? p_first + n_tok - a.window : 0;
      float m_used = -INFINITY, l = 0.f;
      bool any = false;
      for (int i = i0; i < i1; ++i, ++kv) {
        const int kt = ck_tile(t, i), k0 = kt * 128;
        if (!ck_active(a, t, wt, kt)) continue;
        const bool masked = k0 + 128 > full_hi || (k0 < full_lo && k0 + 128 > a.sinks);
        if (!wait_all(s_full(wt), n_s & 1, 0x68)) return false;
        ++n_s;
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tSt + c * 32, sv[c]);
        tmem_wait_ld();
        if (masked) {
          // key k0 + x is visible for x < up, and x >= down or x < top; every other score becomes -inf. One bit mask per
          // 32 keys: this path runs rarely, so its length (cold instruction cache) counts for more than its arithmetic.
          const int up = hi - k0, down = a.window > 0 ? lo - k0 : 0, top = a.sinks - k0;
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t vis = below(up - 32 * c) & (~below(down - 32 * c) | below(top - 32 * c));
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[c][e] = (vis >> e) & 1 ? sv[c][e] : 0xFF800000u;
          }
          // V rows that no row of the pair sees (such tiles are masked ones)
          if (k0 + 128 > t.hi || (k0 < t.lo && k0 + 128 > a.sinks)) {
            const int key = k0 + r;
            const uint32_t st = kv % NST;
            if (!wait_all(v_full(st), (kv / NST) & 1, 0x69)) return false;
            if (key >= t.hi || (key < t.lo && key >= a.sinks)) {
#pragma unroll
              for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sV(st) + h * CK_HALF + r * 128 + u * 16), "r"(0)
                               : "memory");
            }
            fence_proxy_async_smem();
          }
        }
        float mxa[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) mxa[u] = fmaxf(__uint_as_float(sv[0][u]), __uint_as_float(sv[0][u + 8]));
#pragma unroll
        for (int x = 16; x < 128; x += 16)
#pragma unroll
          for (int u = 0; u < 8; ++u)
            mxa[u] = fmax3(mxa[u], __uint_as_float(sv[x >> 5][(x & 31) + u]), __uint_as_float(sv[x >> 5][(x & 31) + 8 + u]));
        const float mx = fmaxf(fmax3(mxa[0], mxa[1], mxa[2]), fmax3(fmax3(mxa[3], mxa[4], mxa[5]), mxa[6], mxa[7])) * sl2;
        const float m_new = fmaxf(m_used, mx);
        if (!any) {
          m_used = m_new;
          any = true;
        } else {
          const bool need = m_new > m_used + 8.f;
          if (__any_sync(0xFFFFFFFFu, need)) {
            // s_full was committed after this tile's previous product: O is quiescent
            const float f = need ? exp2f(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t rr[32];
              tmem_ld32(tOt + c * 32, rr);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) rr[e] = __float_as_uint(__uint_as_float(rr[e]) * f);
              tmem_st32(tOt + c * 32, rr);
            }
            l *= f;
            if (need) m_used = m_new;
          }
        }
        const float m_eff = m_used == -INFINITY ? 0.f : m_used;
        // P = exp2(S scale - m) in bf16 (half a step, 2^-8 of each); the row sum is taken before that rounding. All on the
        // MUFU: a polynomial for a part of them on the FMA pipe lengthened the one thread's run that the other tile's
        // products have to cover (0 / 1 / 2 / 3 / 4 of 8 by polynomial: 878 / 898 / 894 / 909 / 933 us for 2048 tokens
        // over 32768 keys).
        const uint64_t sl2_2 = pack_f2(sl2, sl2), negm2 = pack_f2(-m_eff, -m_eff);
        uint64_t ls2[2] = {0ull, 0ull};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t pk[32];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const uint32_t* s8 = &sv[2 * hf + (g >> 2)][8 * (g & 3)];
            uint64_t x[4], p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = ffma2(pack_u2(s8[2 * u], s8[2 * u + 1]), sl2_2, negm2);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float x0, x1;
              unpack_f2(x[u], x0, x1);
              p[u] = pack_f2(exp2f(x0), exp2f(x1));
            }
            ls2[g & 1] = fadd2(ls2[g & 1], fadd2(fadd2(p[0], p[1]), fadd2(p[2], p[3])));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float p0, p1;
              unpack_f2(p[u], p0, p1);
              pk[4 * g + u] = pack_bf16(p0, p1);
            }
          }
          tmem_st32(tSt + hf * 32, pk);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(hf ? p_full(wt) : p_half(wt));
        }
        {
          float s0, s1;
          unpack_f2(fadd2(ls2[0], ls2[1]), s0, s1);
          l += s0 + s1;
        }
      }
      // ---- epilogue of the piece
      if (any) {
        if (!wait_all(o_done(wt), n_o & 1, 0x6A)) return false;
        ++n_o;
        tc_fence_after();
      }
      const bool whole = i0 == 0 && i1 == t.nt;
      if (whole) {
        // 64 columns at a time through shared memory, so that a store instruction writes 4 rows of 128 bytes instead of
        // 32 rows of 16 (rows of o lie H x D elements apart for every token)
        const float inv = l > 0.f ? 1.f / l : 0.f;
        unsigned long long out = 0;  // address of this row of o, 0: no such row
        if (live) out = (unsigned long long)((__nv_bfloat16*)a.o +
                                             ((long long)(q.q0 + t.tok0 + wt * tpt + rt) * a.H + w.hk * G + rg) * D);
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          uint32_t rr[2][32];
          if (any) {
            tmem_ld32(tOt + c * 64, rr[0]);
            tmem_ld32(tOt + c * 64 + 32, rr[1]);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) rr[e >> 5][e & 31] = 0u;
          }
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const uint32_t* x = &rr[g >> 2][(g & 3) * 8];
            uint32_t y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) y[u] = pack_bf16(__uint_as_float(x[2 * u]) * inv, __uint_as_float(x[2 * u + 1]) * inv);
            // piece g of row `lane`; the exclusive or spreads the rows of a quarter warp over the banks
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((g ^ (lane & 7)) << 4)),
                         "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                         : "memory");
          }
          __syncwarp();
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int row = g * 4 + (lane >> 3), piece = lane & 7;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(stage + row * 128 + ((piece ^ (row & 7)) << 4))
                         : "memory");
            const unsigned long long to = __shfl_sync(0xFFFFFFFFu, out, row);
            if (to) *reinterpret_cast<uint4*>(to + c * 128 + piece * 16) = v;
          }
          __syncwarp();
        }
      } else {
        // partial result: vectors of four columns, each for all 256 rows of the pair side by side
        float* slot = ws + (long long)(2 * blockIdx.x + (i0 == 0 ? 1 : 0)) * Cfg::SLOT;
        const int srow = wt * 128 + r;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t rr[32];
          if (any) {
            tmem_ld32(tOt + c * 32, rr);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) rr[e] = 0u;
          }
          if (live) {
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<uint4*>(slot + ((c * 8 + g) * 256 + srow) * 4) =
                  make_uint4(rr[4 * g], rr[4 * g + 1], rr[4 * g + 2], rr[4 * g + 3]);
          }
          __syncwarp();
        }
        if (live) {
          slot[256 * D + srow] = m_used;
          slot[256 * D + 256 + srow] = l;
        }
      }
      tc_fence_before();  // O has been read: the next piece's products, ordered after the next p_half, may overwrite it
      if (!whole && i0 == 0 && threadIdx.x == 128) {
        const long long end_unit = u1 - w.left - w.first + t.nt + CK_ITEM_COST - 1;  // last unit of this item
        long long i = div_nonneg(end_unit * n_blocks, total);           // share it belongs to
        while (i + 1 < n_blocks && share(i + 1) <= end_unit) ++i;
        while (i > 0 && share(i) > end_unit) --i;
        hdr[blockIdx.x] = make_int4(w.seq, w.hk, w.pair, (int)(i - blockIdx.x + 1));
      }
      return true;
    });
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the item that block blockIdx.x began and later blocks went on with: a thread per row of the pair,
// blockIdx.y takes 8 columns.
template <int D>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const LbPagedAttnArgs a, const float* ws, const int4* hdr) {
  using Cfg = CkCfg<D>;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 h = hdr[blockIdx.x];
  if (h.w == 0) return;
  const int G = a.H / a.Hkv, tpt = 128 / G;
  const CkSeq q = ck_seq(a, h.x, false);
  const int row = threadIdx.x, r = row & 127, tok = h.z * 2 * tpt + (row >> 7) * tpt + r / G;
  if (r >= tpt * G || tok >= q.nq) return;
  auto slot = [&](int part) { return ws + (long long)(part == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + part)) * Cfg::SLOT; };
  float m = -INFINITY, l = 0.f;
  float4 o[2];
  o[0] = o[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int part = 0; part < h.w; part += 4) {  // four parts' loads in flight
    float pm[4], pl[4];
    float4 x[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* p = slot(min(part + u, h.w - 1));
      pm[u] = part + u < h.w ? p[256 * D + row] : -INFINITY;
      pl[u] = p[256 * D + 256 + row];
#pragma unroll
      for (int g = 0; g < 2; ++g) x[u][g] = *reinterpret_cast<const float4*>(p + ((blockIdx.y * 2 + g) * 256 + row) * 4);
    }
    const float mn = fmaxf(m, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])));
    const float f0 = m == -INFINITY ? 0.f : exp2f(m - mn);
    m = mn;
    l *= f0;
#pragma unroll
    for (int g = 0; g < 2; ++g) { o[g].x *= f0; o[g].y *= f0; o[g].z *= f0; o[g].w *= f0; }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = pm[u] == -INFINITY ? 0.f : exp2f(pm[u] - mn);
      l += f * pl[u];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        o[g].x += f * x[u][g].x; o[g].y += f * x[u][g].y; o[g].z += f * x[u][g].z; o[g].w += f * x[u][g].w;
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<uint4*>((__nv_bfloat16*)a.o + ((long long)(q.q0 + tok) * a.H + h.y * G + r % G) * D + blockIdx.y * 8) =
      make_uint4(pack_bf16(o[0].x * inv, o[0].y * inv), pack_bf16(o[0].z * inv, o[0].w * inv),
                 pack_bf16(o[1].x * inv, o[1].y * inv), pack_bf16(o[1].z * inv, o[1].w * inv));
}

template <int D>
static int launch_chunk(const LbPagedAttnArgs& a, void* ws, cudaStream_t st) {
  using Cfg = CkCfg<D>;
  if (ensure_dyn_smem<paged_chunk_kernel<D>>(Cfg::SMEM)) return 20;
  const int G = a.H / a.Hkv, rows = a.page < 128 ? a.page : 128;
  CUtensorMap tq, tk, tv;
  // q as (channel, head, token): a box is the group's heads of as many tokens as make up 128 rows
  const long long qd[4] = {D, a.H, a.T, 1}, qs[3] = {a.q_sh, a.q_st, a.q_st * a.T};
  const int qb[4] = {64, G, 128 / G, 1};
  if (make_tmap_box(&tq, a.q, 2, qd, qs, qb)) return 9;
  if (make_tmap_4d(&tk, a.k_pages, 2, D, a.page, a.kp_st, a.Hkv, a.kp_sh, a.n_pages, a.kp_sp, 64, rows)) return 10;
  if (make_tmap_4d(&tv, a.v_pages, 2, D, a.page, a.vp_st, a.Hkv, a.vp_sh, a.n_pages, a.vp_sp, 64, rows)) return 11;
  const int grid = num_sms();
  int4* hdr = reinterpret_cast<int4*>((float*)ws + 2ll * grid * Cfg::SLOT);
  paged_chunk_kernel<D><<<grid, CK_THREADS, Cfg::SMEM, st>>>(tq, tk, tv, a, (float*)ws, hdr);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, D / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, paged_chunk_join_kernel<D>, a, (const float*)ws, (const int4*)hdr) != cudaSuccess)
    return 400 + (int)cudaGetLastError();
  g_launches.fetch_add(1, std::memory_order_relaxed);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

long long paged_chunk_workspace(int D) {
  return (long long)num_sms() * (2ll * (D == 128 ? CkCfg<128>::SLOT : CkCfg<64>::SLOT) * 4 + 16);
}
int paged_chunk_dispatch(const LbPagedAttnArgs& a, void* ws, cudaStream_t st) {
  return a.D == 128 ? launch_chunk<128>(a, ws, st) : launch_chunk<64>(a, ws, st);
}

}  // namespace lb
