// Attention of few new tokens per sequence over a paged KV cache (see paged_cache.cu for the layout of cache and batch).
//
// The query of a token at position p sees the keys j <= p of its sequence and, with a sliding window W, of those only
// the ones with j > p - W or j < sinks. A row that sees no key (a padding row, an empty sequence) gives zeros.
//
// Bound by reading every visible key and value row once (2 D 2 bytes per key and kv head; G = H / Hkv query heads share
// them). Measured: 64 sequences of up to 8192 keys, 32 / 8 heads (1.2 GB) 188 us, 6.4 TB/s; one of 131072 keys 90 us, 6.0 TB/s;
// one of 511 keys, 16 heads, 6.6 us (in a graph). Layout of the work:
//  * An item is (sequence, kv head, 8 or 16 rows), the rows being (token, head of the group) pairs, so that one pass over
//    the keys serves the whole group. The products are m16n8k16 with the KEYS on the 16 side and the rows on the 8 side,
//    S^T = K Q^T and O^T = V^T P^T: with the rows on the 16 side, as one would write them first, one token of up to 8
//    heads would fill half of every product.
//  * The key axis of an item is cut into blocks of 64 keys. All blocks of all items, in order, are dealt out in equal
//    contiguous shares to the blocks of a fixed grid, so a batch of any mix of lengths keeps every SM equally busy; an
//    item that crosses a share boundary leaves partial results (running maximum, sum, unnormalised output, fp32) that
//    a second small kernel joins. The shares follow from the lengths on the device: a captured graph can be replayed with
//    other lengths. When the table's width allows no item longer than NOSPLIT_BLOCKS blocks, items are dealt out whole
//    instead and the second kernel is not launched. A few sequences of moderate length (one token each) are cut by
//    clusters: up to 8 blocks share an item and join their parts through distributed shared memory, in one launch.
//  * The four warps of a block take 16 keys of a 64-key block each and meet only at the end of an item. Every warp
//    keeps its own ring of 16-key stages in shared memory, filled by TMA (boxes of 16 keys x 64 channels, 128-byte
//    swizzle), so a stage is waited for and given back by one warp alone. The join at the end of an item takes one stage of
//    each ring (two for 16 rows); the others fill with the next item's first blocks meanwhile (batch below 196 -> 188 us).
//  * ldmatrix reads both operands in place, the values transposed; the swizzle makes its eight rows fall into different
//    banks. P^T is turned from the layout of a result to that of an operand by movmatrix.
//  * Keys that no row may see, and pages that are not there, never contribute: scores are replaced (not added to), and
//    values of hidden keys are zeroed in registers, so what a page holds past the end of a sequence (NaN included)
//    or behind the window does not matter.
#include <algorithm>
#include "common.cuh"
#include "lingua_b200.h"

namespace lb {

constexpr int DEC_BLOCK = 64;       // keys per block: 16 for each warp
// Items of up to so many blocks are not cut up into shares that a second kernel joins: 256 keys 7.4 us whole,
// 300 keys 8.4 us whole and 8.0 us cut up, 511 keys 10.6 / 8.0 (one sequence, 16 heads, in a graph).
constexpr int NOSPLIT_BLOCKS = 4;
constexpr float DEC_LOG2E = 1.4426950408889634f;

template <int D, int NT>
struct DecCfg {
  static constexpr int ROWS = 8 * NT;
  static constexpr int VG = D / 64;            // 64-channel boxes of a row
  static constexpr int BOX = 16 * 128;         // 16 keys x 64 channels
  static constexpr int STAGE = 2 * VG * BOX;   // bytes of one warp's stage: key boxes, then value boxes
  static constexpr int NST = D == 128 ? 3 : 6;
  static constexpr int SMEM = 4 * NST * STAGE + 1024;  // 97 KB: two blocks per SM
  static constexpr int OROW = D + 4;                // padded row of the merge buffer (floats)
  static_assert(8 * OROW * 4 <= STAGE && NT < NST, "a stage holds a row tile of the merge buffer");
  static constexpr int SLOT = ROWS * D + 2 * ROWS;  // floats of one partial result
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&m)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&m)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_cluster(uint32_t saddr, int rank) {  // the same address in block `rank`'s shared memory
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a)
               : "memory");
  return v;
}

// What a sequence asks for.
struct DecSeq {
  int q0, nq;       // its rows of q
  long long pos0;   // position of its first new token (may be negative)
  int end;          // visible keys end here
  int wlo;          // first key inside some row's window
  int sb, wb;       // 64-key blocks: [0, sb) for the first tokens, then from wb on
  int nb;           // blocks of an item (at least one: rows that see nothing still get their zeros)
  int rt;           // row tiles
};

template <int ROWS>
__device__ __forceinline__ DecSeq dec_seq(const LbPagedAttnArgs& a, int s, bool report) {
  DecSeq r;
  r.q0 = a.cu_q ? a.cu_q[s] : s;
  r.nq = a.cu_q ? a.cu_q[s + 1] - r.q0 : 1;
  const int cap = a.cols * a.page;
  const int len = a.kv_len[s];
  if (report && len > cap && a.status) atomicOr(a.status, ST_BAD_ARG | 0x43u);
  if (r.q0 < 0 || r.nq < 0 || r.q0 > a.T - r.nq) {  // rows that q does not have
    if (report && a.status) atomicOr(a.status, ST_BAD_ARG | 0x45u);
    r.nq = 0;
  }
  r.pos0 = (long long)len - r.nq;
  r.end = max(0, min(len, cap));
  r.wlo = 0;
  if (a.window > 0) r.wlo = (int)max(0ll, min((long long)r.end, r.pos0 - a.window + 1));
  r.wb = r.wlo / DEC_BLOCK;
  r.sb = min((min(a.sinks, r.wlo) + DEC_BLOCK - 1) / DEC_BLOCK, r.wb);
  r.nb = max(1, r.sb + (r.end + DEC_BLOCK - 1) / DEC_BLOCK - r.wb);
  const long long rows = (long long)r.nq * (a.H / a.Hkv);
  r.rt = (int)((rows + ROWS - 1) / ROWS);
  return r;
}

// A block's part of an item: kv head, row tile and 64-key blocks [b0, b1) of a sequence.
struct DecPiece {
  int seq, hk, rt, b0, b1;
  DecSeq q;
};

struct DecWork {  // found by one thread, read by the block
  int seq;           // sequence of this block's first unit
  long long offset;  // units of that sequence before it
};

// Workspace: per block two partial results (its first item when an earlier block began it, its last item when a later
// block ends it) and one int4 header naming the item it began without ending: (sequence, kv head, row tile, parts).
template <int D, int NT>
__global__ void __launch_bounds__(128, 2) paged_decode_kernel(const __grid_constant__ CUtensorMap tk,
                                                              const __grid_constant__ CUtensorMap tv,
                                                              const LbPagedAttnArgs a, float* ws, int4* hdr, int cl) {
  using Cfg = DecCfg<D, NT>;
  constexpr int ROWS = Cfg::ROWS;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[4][Cfg::NST];
  __shared__ int abort_flag;
  __shared__ long long warp_sum[4];
  __shared__ DecWork work;
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  __shared__ float part_m[ROWS], part_l[ROWS];  // of this block's part of a cluster's item
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int G = a.H / a.Hkv;
  const bool split = ws != nullptr || cl;  // cl: blocks of a cluster that share an item, 0 without clusters
  const uint32_t dyn0 = (smem_u32(dyn) + 1023u) & ~1023u;  // the swizzle pattern repeats every 1024 bytes
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int w = 0; w < 4; ++w)
      for (int st = 0; st < Cfg::NST; ++st) mbar_init(smem_u32(&full[w][st]), 1);
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this block's share: a unit is one 64-key block of an item (or a whole item without splitting)
  long long u0, u1, total = 0, n_blocks = 1;
  auto share = [&](long long i) { return div_nonneg(total * i, n_blocks); };  // first unit of share i
  if (cl) {
    const int item = blockIdx.x / cl, rank = blockIdx.x % cl, per_seq = gridDim.x / (a.n_seqs * cl);
    const int s = item / per_seq;
    const DecSeq q = dec_seq<ROWS>(a, s, rank == 0 && item % per_seq == 0);
    u0 = (long long)q.nb * rank / cl;
    u1 = (long long)q.nb * (rank + 1) / cl;
    if (threadIdx.x == 0) { work.seq = s; work.offset = (long long)(item % per_seq) * q.nb + u0; }
    if (threadIdx.x < ROWS) { part_m[threadIdx.x] = -INFINITY; part_l[threadIdx.x] = 0.f; }
  } else {
  const int per = (a.n_seqs + 127) / 128;
  const int s_lo = min(a.n_seqs, (int)threadIdx.x * per), s_hi = min(a.n_seqs, s_lo + per);
  long long mine = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const DecSeq q = dec_seq<ROWS>(a, s, blockIdx.x == 0);
    mine += (long long)a.Hkv * q.rt * (split ? q.nb : 1);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  long long before = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  before += incl - mine;
  // no share is empty (the join kernel counts on that)
  n_blocks = max(1ll, min((long long)gridDim.x, total));
  const bool busy = blockIdx.x < n_blocks;
  u0 = busy ? share(blockIdx.x) : 0;
  u1 = busy ? share(blockIdx.x + 1) : 0;
  if (u0 < u1 && u0 >= before && u0 < before + mine) {
    long long at = before;
    for (int s = s_lo; s < s_hi; ++s) {
      const DecSeq q = dec_seq<ROWS>(a, s, false);
      const long long n = (long long)a.Hkv * q.rt * (split ? q.nb : 1);
      if (u0 < at + n) { work.seq = s; work.offset = u0 - at; break; }
      at += n;
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
      for (long long i = threadIdx.x; i < vec; i += 128) row[i] = make_uint4(0, 0, 0, 0);
    }
  }
  if (hdr && threadIdx.x == 0) hdr[blockIdx.x] = make_int4(0, 0, 0, 0);
  __syncthreads();
  if (u0 >= u1 && !cl) return;

  const uint32_t ring = dyn0 + warp * (Cfg::NST * Cfg::STAGE);
  const uint32_t bars = smem_u32(&full[warp][0]);
  uint32_t parity = 0;  // bit st: phase the next wait on stage st completes
  int head = 0;         // stage of the next block to be read
  bool alive = true;
  // ldmatrix row of this lane: matrix lane >> 3, row lane & 7. Keys: matrices (keys 0-7, piece), (keys 8-15, piece), then the
  // next piece; values: (keys 0-7, piece), (keys 0-7, next piece), then keys 8-15. Offsets of pieces 2 p, 2 p + 1 of a box.
  const int k_row = (lane & 7) + 8 * ((lane >> 3) & 1), v_row = (lane & 7) + 8 * (lane >> 4);
  uint32_t k_off[4], v_off[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    k_off[p] = k_row * 128 + (((2 * p + (lane >> 4)) ^ (lane & 7)) << 4);
    v_off[p] = v_row * 128 + (((2 * p + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
  }
  const float sl2 = a.scale * DEC_LOG2E;
  const int page_log = __ffs(a.page) - 1;
  // pieces of this block's share, one after the other
  long long left = u1 - u0, item = 0, n_items = 0;
  int first = 0;  // key block that the next piece begins with
  DecPiece nxt;
  nxt.seq = work.seq;
  auto enter = [&]() {
    nxt.q = dec_seq<ROWS>(a, nxt.seq, false);
    n_items = (long long)a.Hkv * nxt.q.rt;
  };
  auto fetch = [&]() {
    while (left > 0) {
      if (item < n_items) {
        nxt.hk = (int)div_nonneg(item, nxt.q.rt);
        nxt.rt = (int)(item - (long long)nxt.hk * nxt.q.rt);
        nxt.b0 = first;
        nxt.b1 = split ? (int)min((long long)nxt.q.nb, first + left) : nxt.q.nb;
        left -= split ? nxt.b1 - nxt.b0 : 1;
        first = 0;
        ++item;
        return true;
      }
      if (++nxt.seq >= a.n_seqs) return false;
      item = 0;
      enter();
    }
    return false;
  };
  enter();
  item = div_nonneg(work.offset, split ? nxt.q.nb : 1);
  if (split) first = (int)(work.offset - item * nxt.q.nb);

  // ---- requests: pages of a piece's next 32 + 32 blocks, one per lane
  int pg = -1, pg_next = -1, filled = 0;
  auto key_of = [&](const DecPiece& w, int b) { return (b < w.q.sb ? b : b - w.q.sb + w.q.wb) * DEC_BLOCK + warp * 16; };
  auto page_of = [&](const DecPiece& w, int b) {
    const int k = key_of(w, b);
    return b < w.b1 && k < w.q.end ? __ldg(a.table + (long long)w.seq * a.table_stride + (k >> page_log)) : -1;
  };
  auto issue = [&](const DecPiece& w, int b, int st) {
    const int rel = b - w.b0;
    if ((rel & 31) == 0 && rel) pg = pg_next;
    if ((rel & 31) == 16) pg_next = page_of(w, b + 16 + lane);
    int page = __shfl_sync(0xFFFFFFFFu, pg, rel & 31);
    if (lane == 0) {
      const int kb = key_of(w, b), off = kb & (a.page - 1);
      // 16 keys that no row sees are requested outside the pool, where TMA fills with zeros and reads nothing (with a window
      // of 1024 and the first 4 keys that is a tenth of the bytes: 48 sequences of 32 heads 138 -> 130 us). A visible key
      // without a page is an error.
      const bool seen = kb < w.q.end && (kb + 16 > w.q.wlo || kb < a.sinks);
      if (!seen) page = a.n_pages;
      if (page < 0 || page >= a.n_pages) {
        if (seen && a.status) atomicOr(a.status, ST_BAD_ARG | 0x44u);
        page = a.n_pages;
      }
      const uint32_t bar = bars + 8 * st, dst = ring + st * Cfg::STAGE;
      mbar_arrive_expect_tx(bar, Cfg::STAGE);
#pragma unroll
      for (int g = 0; g < Cfg::VG; ++g) tma_load_4d(dst + g * Cfg::BOX, &tk, bar, 64 * g, off, w.hk, page);
#pragma unroll
      for (int g = 0; g < Cfg::VG; ++g) tma_load_4d(dst + (Cfg::VG + g) * Cfg::BOX, &tv, bar, 64 * g, off, w.hk, page);
    }
  };
  auto wrap = [](int st) { return st >= Cfg::NST ? st - Cfg::NST : st; };
  // the first blocks of the next piece, until n stages are filled (all are free once a piece's blocks have been read)
  auto fill = [&](int n) {
#pragma unroll 1
    for (; filled < min(nxt.b1 - nxt.b0, n); ++filled) issue(nxt, nxt.b0 + filled, wrap(head + filled));
  };

  bool have = fetch();
  if (have) pg = page_of(nxt, nxt.b0 + lane);
  while (have) {
    const DecPiece w = nxt;
    const DecSeq& q = w.q;
    const int hk = w.hk, b0 = w.b0, b1 = w.b1;

    // ---- Q^T fragments: lane (r, c) holds channels 16 k + 2 c, + 1, + 8, + 9 of row 8 t + r
    const int row0 = w.rt * ROWS;
    const int n_rows = min(ROWS, q.nq * G - row0);
    uint32_t qf[D / 16][NT][2];
    long long pos[NT][2];  // of rows 8 t + 2 c, + 1
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = row0 + 8 * t + r;
      const bool live = 8 * t + r < n_rows;
      const __nv_bfloat16* qp = (const __nv_bfloat16*)a.q + (long long)(q.q0 + row / G) * a.q_st +
                                (long long)(hk * G + row % G) * a.q_sh + 2 * c;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][t][0] = live ? *reinterpret_cast<const uint32_t*>(qp + 16 * k) : 0u;
        qf[k][t][1] = live ? *reinterpret_cast<const uint32_t*>(qp + 16 * k + 8) : 0u;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pos[t][i] = 8 * t + 2 * c + i < n_rows ? q.pos0 + (row0 + 8 * t + 2 * c + i) / G : -1;
    }

    fill(Cfg::NST);  // of what the previous piece's end has left
    filled = 0;

    // rows 8 t + 2 c + i: maximum, sum, and O^T: acc[j][t][2 h + i] is channel 16 j + 8 h + r
    float m[NT][2], l[NT][2];
    float acc[D / 16][NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) { m[t][i] = -INFINITY; l[t][i] = 0.f; }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][t][i] = 0.f;
    }

    int prev = head;
    for (int b = b0; alive && b < b1; ++b) {
      alive = mbar_wait(bars + 8 * head, (parity >> head) & 1, &abort_flag, a.status, 0x46);
      alive = __all_sync(0xFFFFFFFFu, alive);
      if (!alive) break;
      parity ^= 1u << head;
      const uint32_t kbox = ring + head * Cfg::STAGE, vbox = kbox + Cfg::VG * Cfg::BOX;
      // scores: two accumulators for each row tile, so that chains of dependent products are half as long
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = s2[t][i] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t kf[4];
        ldmatrix_x4(kf, kbox + (k >> 2) * Cfg::BOX + k_off[k & 3]);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816(k & 1 ? s2[t] : s[t], kf, qf[k][t][0], qf[k][t][1]);
      }
      // what follows needs time until the scores are there: refill the stage of the previous block, read the values
      if (b > b0 && b + Cfg::NST - 1 < b1) issue(w, b + Cfg::NST - 1, prev);
      uint32_t vf[D / 16][4];
#pragma unroll
      for (int j = 0; j < D / 16; ++j) ldmatrix_x4_trans(vf[j], vbox + (j >> 2) * Cfg::BOX + v_off[j & 3]);
      // in units of log 2; s[t][2 h + i]: key kb + r + 8 h, row 8 t + 2 c + i
      const int kb = key_of(w, b);
      const bool whole = kb + 16 <= q.end - (q.nq - 1) && (kb > q.end - 1 - a.window || a.window <= 0 || kb + 16 <= a.sinks);
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          s[t][x] = (s[t][x] + s2[t][x]) * sl2;
          if (!whole) {
            const int j = kb + r + 8 * (x >> 1);
            const long long p = pos[t][x & 1];
            if (j > p || j >= q.end || (a.window > 0 && j <= p - a.window && j >= a.sinks)) s[t][x] = -INFINITY;
          }
        }
        // the running maximum only moves when it would be exceeded by more than 2^8 (probabilities stay below 2^8)
#pragma unroll
        for (int i = 0; i < 2; ++i) grow |= fmaxf(s[t][i], s[t][2 + i]) > m[t][i] + 8.f;
      }
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(s[t][i], s[t][2 + i]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
            if (mx > m[t][i]) {
              const float f = m[t][i] == -INFINITY ? 0.f : exp2f(m[t][i] - mx);
              m[t][i] = mx;
              l[t][i] *= f;
#pragma unroll
              for (int j = 0; j < D / 16; ++j) { acc[j][t][i] *= f; acc[j][t][2 + i] *= f; }
            }
          }
      }
      // probabilities enter the second product in bf16 (half a step, 2^-8 of each); their sum is taken before that
      uint32_t pt[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float m0 = m[t][0] == -INFINITY ? 0.f : m[t][0], m1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = exp2f(s[t][2 * h] - m0), p1 = exp2f(s[t][2 * h + 1] - m1);
          l[t][0] += p0;
          l[t][1] += p1;
          pt[t][h] = movmatrix_trans(pack_bf16(p0, p1));
        }
      }
      uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;  // keys kb + 2 c, + 1 and those 8 further: which are not hidden
      if (!whole) {
        keep0 = keep1 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = kb + 2 * c + (i & 1) + 8 * (i >> 1);
          const uint32_t bits = j < q.end && (j >= q.wlo || j < a.sinks) ? 0xFFFFu << (16 * (i & 1)) : 0u;
          if (i < 2) keep0 |= bits; else keep1 |= bits;
        }
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        if (!whole) { vf[j][0] &= keep0; vf[j][1] &= keep0; vf[j][2] &= keep1; vf[j][3] &= keep1; }
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816(acc[j][t], vf[j], pt[t][0], pt[t][1]);
      }
      __syncwarp();  // every lane's pieces are in registers (the products needed them): the stage can be filled again
      prev = head;
      head = wrap(head + 1);
    }
    // ---- join the four warps. The last NT stages of each ring, counted from where the next piece begins, hold its partial
    // output; the others take the next piece's first blocks meanwhile.
    have = left > 0 && fetch();
    if (have && alive) {
      pg = page_of(nxt, nxt.b0 + lane);
      fill(Cfg::NST - NT);
    }
    auto obuf = [&](int of, int row) {  // of a cluster's block: where its neighbours know it to be
      const int st = cl ? row >> 3 : wrap(head + Cfg::NST - 1 - (row >> 3));
      return reinterpret_cast<float*>(dyn + (dyn0 - smem_u32(dyn)) + (of * Cfg::NST + st) * Cfg::STAGE) + (row & 7) * Cfg::OROW;
    };
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], o);
        if (r == 0) { sm_m[warp][8 * t + 2 * c + i] = m[t][i]; sm_l[warp][8 * t + 2 * c + i] = l[t][i]; }
      }
    __syncthreads();
    if (abort_flag) {  // a wait ran out (recorded in the status word); read by all after the same barrier
      // copies in flight land before shared memory is given up
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
      if (!cl) return;
      break;  // the other blocks of the cluster are met below; this one has nothing to add
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 8 * t + 2 * c + i;
        if (row < n_rows) {
          const float M = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row]));
          const float f = m[t][i] == -INFINITY ? 0.f : exp2f(m[t][i] - M);
          float* dst = obuf(warp, row) + r;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            dst[16 * j] = acc[j][t][i] * f;
            dst[16 * j + 8] = acc[j][t][2 + i] * f;
          }
        }
      }
    __syncthreads();
    const bool whole_item = b0 == 0 && b1 == q.nb;
    float* slot = whole_item || cl ? nullptr : ws + (long long)(2 * blockIdx.x + (b0 == 0 ? 1 : 0)) * Cfg::SLOT;
    for (int i = threadIdx.x; i < n_rows * (D / 4); i += 128) {
      const int row = i / (D / 4), ch = (i % (D / 4)) * 4;
      const float M = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row]));
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
#pragma unroll
      for (int of = 0; of < 4; ++of) {
        const float4 x = *reinterpret_cast<const float4*>(obuf(of, row) + ch);
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
        L += sm_l[of][row] == 0.f ? 0.f : sm_l[of][row] * exp2f(sm_m[of][row] - M);  // NaN scores leave m at -inf
      }
      if (cl) {  // nobody else reads or writes these four floats of the merge buffer
        *reinterpret_cast<float4*>(obuf(0, row) + ch) = o;
        if (ch == 0) { part_m[row] = M; part_l[row] = L; }
      } else if (whole_item) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int gr = row0 + row;
        __nv_bfloat16* op = (__nv_bfloat16*)a.o + ((long long)(q.q0 + gr / G) * a.H + hk * G + gr % G) * D + ch;
        *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      } else {
        *reinterpret_cast<float4*>(slot + row * D + ch) = o;
        if (ch == 0) { slot[ROWS * D + row] = M; slot[ROWS * D + ROWS + row] = L; }
      }
    }
    if (cl) break;
    if (!whole_item && b0 == 0 && threadIdx.x == 0) {
      // units [u1 - (b1 - b0), + nb) hold this item: find the block its last unit belongs to
      const long long end_unit = u1 - (b1 - b0) + q.nb - 1;
      // share of unit u: the largest i with total * i / n_blocks <= u
      long long i = div_nonneg(end_unit * n_blocks, total);
      while (i + 1 < n_blocks && share(i + 1) <= end_unit) ++i;
      while (i > 0 && share(i) > end_unit) --i;
      hdr[blockIdx.x] = make_int4(w.seq, hk, w.rt, (int)(i - blockIdx.x + 1));
    }
    fence_proxy_async_smem();  // the merge buffer becomes the ring again: ordinary accesses before TMA writes
    __syncthreads();
  }
  if (!cl) return;

  // ---- join the cluster's parts: every block is met here, whatever became of its part, and each writes a slice
  cluster_sync();
  {
    const int item = blockIdx.x / cl, rank = blockIdx.x % cl, per_seq = gridDim.x / (a.n_seqs * cl);
    const DecSeq q = dec_seq<ROWS>(a, item / per_seq, false);
    const int hk = (item % per_seq) / q.rt, row0 = (item % per_seq) % q.rt * ROWS;
    const int n_rows = min(ROWS, q.nq * G - row0);
    const uint32_t pm = smem_u32(part_m), pl = smem_u32(part_l);
    for (int i = threadIdx.x + 128 * rank; i < n_rows * (D / 4); i += 128 * cl) {
      const int row = i / (D / 4), ch = (i % (D / 4)) * 4;
      // all parts' loads in flight at once; the buffer of a part that saw no key may hold anything
      float m[8], l[8], M = -INFINITY, L = 0.f;
      float4 x[8], o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        m[p] = -INFINITY;
        l[p] = 0.f;
        if (p < cl) {
          m[p] = ld_cluster(map_cluster(pm + 4 * row, p));
          l[p] = ld_cluster(map_cluster(pl + 4 * row, p));
          x[p] = ld_cluster4(map_cluster(dyn0 + (row >> 3) * Cfg::STAGE + 4 * ((row & 7) * Cfg::OROW + ch), p));
        }
      }
#pragma unroll
      for (int p = 0; p < 8; ++p) M = fmaxf(M, m[p]);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (l[p] != 0.f) {
          const float f = exp2f(m[p] - M);
          L += f * l[p];
          o.x += f * x[p].x; o.y += f * x[p].y; o.z += f * x[p].z; o.w += f * x[p].w;
        }
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int gr = row0 + row;
      __nv_bfloat16* op = (__nv_bfloat16*)a.o + ((long long)(q.q0 + gr / G) * a.H + hk * G + gr % G) * D + ch;
      *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
  }
  cluster_sync();  // nobody leaves while its shared memory is being read
}

// Joins the parts of the item that block `blockIdx.x` of the kernel above began and later blocks went on with: warps
// take parts, lanes channels.
template <int D, int NT>
__global__ void __launch_bounds__(256) paged_decode_join_kernel(const LbPagedAttnArgs a, const float* ws, const int4* hdr) {
  using Cfg = DecCfg<D, NT>;
  constexpr int ROWS = Cfg::ROWS;
  constexpr int E = D / 32;
  __shared__ float sm_o[8][D], sm_m[8], sm_l[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 h = hdr[blockIdx.x];
  if (h.w == 0) return;
  const DecSeq q = dec_seq<ROWS>(a, h.x, false);
  const int G = a.H / a.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = h.z * ROWS + blockIdx.y;
  if (row >= q.nq * G) return;
  auto slot = [&](int part) { return ws + (long long)(part == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + part)) * Cfg::SLOT; };
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int part = warp; part < h.w; part += 8) {
    const float* p = slot(part);
    const float pm = p[ROWS * D + blockIdx.y], pl = p[ROWS * D + ROWS + blockIdx.y];
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = p[blockIdx.y * D + lane * E + e];
    const float mn = fmaxf(m, pm);
    const float fa = m == -INFINITY ? 0.f : exp2f(m - mn), fb = pm == -INFINITY ? 0.f : exp2f(pm - mn);
    m = mn;
    l = l * fa + pl * fb;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * fa + x[e] * fb;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sm_o[warp][lane * E + e] = o[e];
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) M = fmaxf(M, sm_m[w]);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float f = sm_m[w] == -INFINITY ? 0.f : exp2f(sm_m[w] - M);
      L += sm_l[w] * f;
      x += sm_o[w][threadIdx.x] * f;
    }
    ((__nv_bfloat16*)a.o)[((long long)(q.q0 + row / G) * a.H + h.y * G + row % G) * D + threadIdx.x] =
        __float2bfloat16(L == 0.f ? 0.f : x / L);  // 0: the row sees no key. NaN stays NaN
  }
}

template <int D, int NT>
static int launch_decode(const LbPagedAttnArgs& a, void* ws, int cl, cudaStream_t st) {
  using Cfg = DecCfg<D, NT>;
  if (ensure_dyn_smem<paged_decode_kernel<D, NT>>(Cfg::SMEM)) return 20;
  const int grid = 2 * num_sms();
  int4* hdr = ws ? reinterpret_cast<int4*>((float*)ws + 2ll * grid * Cfg::SLOT) : nullptr;
  // pools as (channel, row of the page, head, page), read in boxes of 64 channels x 16 rows
  CUtensorMap tk, tv;
  if (make_tmap_4d(&tk, a.k_pages, 2, D, a.page, a.kp_st, a.Hkv, a.kp_sh, a.n_pages, a.kp_sp, 64, 16)) return 10;
  if (make_tmap_4d(&tv, a.v_pages, 2, D, a.page, a.vp_st, a.Hkv, a.vp_sh, a.n_pages, a.vp_sp, 64, 16)) return 11;
  if (cl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_seqs * a.Hkv * ((a.H / a.Hkv + Cfg::ROWS - 1) / Cfg::ROWS) * cl);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cl;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, NT>, tk, tv, a, (float*)nullptr, (int4*)nullptr, cl);
    if (e != cudaSuccess) return 400 + (int)e;
  } else {
    paged_decode_kernel<D, NT><<<grid, 128, Cfg::SMEM, st>>>(tk, tv, a, (float*)ws, hdr, 0);
  }
  g_launches.fetch_add(1, std::memory_order_relaxed);
  if (ws) {
    // starts while the first kernel's last blocks run, and waits for all of it before it reads
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, a.cu_q ? Cfg::ROWS : std::min(Cfg::ROWS, a.H / a.Hkv));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, paged_decode_join_kernel<D, NT>, a, (const float*)ws, (const int4*)hdr) != cudaSuccess) {
      return 400 + (int)cudaGetLastError();
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

}  // namespace lb

namespace lb {
// The few-token kernel passes over a sequence's keys once for every 16 rows (new tokens x heads of a group), the tcgen05
// kernel once for 256. Measured (8 kv heads, 128 channels, us in a graph, few-token / tcgen05): 16 rows 34 / 42 (1 sequence
// of 32768 keys), 331 / 365 (64 of 8192), 105 / 149 (256 of 500); 32 rows 52 / 41, 629 / 367, 180 / 150. With little work for
// each block the few-token kernel's shorter start decides: 1 sequence of 2000 keys 14 / 20 at 32 rows, 20 / 20 at 64,
// 23 / 21 at 128; 300 keys 12 / 15.
constexpr int CHUNK_ROWS = 16;
constexpr int FEW_BLOCKS = 8;  // 64-key blocks for a thread block of the few-token kernel
static bool use_chunk(const LbPagedAttnArgs& a) {
  const int G = a.H / a.Hkv;
  const long long rows = (long long)a.max_q * G;
  if (!a.cu_q || G > 128 || rows <= CHUNK_ROWS) return false;
  const long long blocks = (long long)a.n_seqs * a.Hkv * ((rows + 15) / 16) *
                           (((long long)a.cols * a.page + DEC_BLOCK - 1) / DEC_BLOCK);
  return blocks > 2ll * num_sms() * FEW_BLOCKS;
}
// one row tile of 8 where that holds all rows of a sequence, else of 16
static bool eight_rows(const LbPagedAttnArgs& a) { return (long long)(a.cu_q ? a.max_q : 1) * (a.H / a.Hkv) <= 8; }
// most 64-key blocks an item can have
static long long most_blocks(const LbPagedAttnArgs& a) {
  long long keys = (long long)a.cols * a.page;
  if (a.window > 0 && !a.cu_q) keys = std::min(keys, (long long)a.window + a.sinks + DEC_BLOCK);
  return (keys + DEC_BLOCK - 1) / DEC_BLOCK;
}
// Blocks of a cluster that share an item; 0: no clusters. For one token per sequence, and as long as a block of the
// cluster has no more than FEW_BLOCKS key blocks and the clusters fit the GPU side by side; beyond that equal shares of
// everything are worth the second launch. As many blocks as key blocks, rounded up: a block without keys costs more than it
// gives (16 heads, in a graph, whole / cluster: 128 keys 6.0 / 5.9 us by 2, 6.4 by 8; 256 keys 7.6 / 6.2 by 4, 6.6 by 8;
// 511 keys 10.6 / 6.6 by 8).
static int cluster_size(const LbPagedAttnArgs& a) {
  const long long blocks = most_blocks(a);
  if (a.cu_q || blocks <= 2) return 0;
  const int rows = eight_rows(a) ? 8 : 16;
  const long long items = (long long)a.n_seqs * a.Hkv * ((a.H / a.Hkv + rows - 1) / rows);
  for (int cl = 8; cl > 1; cl /= 2)
    if (cl < 2 * blocks && items * cl <= 2ll * num_sms() && blocks <= (long long)cl * FEW_BLOCKS) return cl;
  return 0;
}
template <int NT>
static long long decode_slot(int D) { return D == 128 ? DecCfg<128, NT>::SLOT : DecCfg<64, NT>::SLOT; }
}  // namespace lb

extern "C" long long lb_paged_attention_workspace(const LbPagedAttnArgs* a) {
  using namespace lb;
  if (use_chunk(*a)) return paged_chunk_workspace(a->D);
  if (most_blocks(*a) <= NOSPLIT_BLOCKS || cluster_size(*a)) return 0;
  const long long slot = eight_rows(*a) ? decode_slot<1>(a->D) : decode_slot<2>(a->D);
  return 2ll * num_sms() * (2 * slot * 4 + 16);
}

extern "C" int lb_paged_attention(const LbPagedAttnArgs* a, void* workspace, void* stream) {
  using namespace lb;
  if (a->D != 64 && a->D != 128) return 1;
  if (a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv) return 2;
  if (a->page < 16 || (a->page & (a->page - 1))) return 3;
  if ((long long)a->cols * a->page > (1ll << 30)) return 4;
  if (a->T <= 0) return 0;
  if (use_chunk(*a)) return workspace ? paged_chunk_dispatch(*a, workspace, (cudaStream_t)stream) : 5;
  cudaStream_t st = (cudaStream_t)stream;
  const int cl = cluster_size(*a);
  if (eight_rows(*a))
    return a->D == 128 ? launch_decode<128, 1>(*a, workspace, cl, st) : launch_decode<64, 1>(*a, workspace, cl, st);
  return a->D == 128 ? launch_decode<128, 2>(*a, workspace, cl, st) : launch_decode<64, 2>(*a, workspace, cl, st);
}
