// attn_decode.cu -- ggufmm_paged_attention: attention of one new token per sequence over
// the paged key-value cache, the cache's length split over the SMs and joined in the same
// launch.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q.k_j,  m = max_j s_j
//
// One pass over the keys and values with a running m and sum. The G = q_heads / kv_heads
// query heads that share a kv head are the rows of one 16-row tensor-core tile, so each
// cached value is read once: 2 G flops per byte, far below what the tensor cores need,
// and the time is the cache's bytes over the HBM rate.
//
// Split: the work is the list of all (sequence, kv head) items, cut into blocks of W * 16
// tokens. Every CTA (one per SM) takes an equal run of consecutive blocks, whatever
// sequences they belong to, so ragged lengths leave no SM idle; it finds its run by a sum
// over the lengths on the device. An item inside one run is written directly. An item that
// crosses runs leaves fp32 partials (m, sum, o) in the workspace, and the last of its CTAs
// to finish (a counter) adds them in the order of the CTAs, so the result does not depend
// on which was last.
//
// Inside a CTA each warp owns every W-th group of 16 tokens and its own ring of stages,
// filled by TMA two pages' worth at a time ahead of use, across items: no barrier between
// warps except where an item ends, and the ring keeps streaming over that too.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "mma16.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace ggufmm {

struct DevInfo {
  int sms = 0;
  int smem_optin = 0;
};
DevInfo device_info(int dev);  // capi.cu

namespace {

constexpr int kMaxGrid = 256;                      // CTAs a workspace has room for
constexpr size_t kCounterBytes = kMaxGrid * 4;     // one arrival counter per CTA that an item may start in

template <int DP>
struct Shape {
  static constexpr int W = DP == 256 ? 4 : 8;       // warps
  static constexpr int NB = DP / 64;                // 128-byte column blocks of a row
  static constexpr int HALF = 16 * DP * 2;          // bytes of 16 tokens of K (or V)
  static constexpr int STAGE = 2 * HALF;
  static constexpr int S = 196608 / (W * STAGE);    // stages per warp
  static constexpr int BLOCK = 16 * W;              // tokens
  static constexpr int RING = W * S * STAGE;
  static constexpr int JOIN = W * 8 * DP * 4;       // 8 rows of every warp's sums
  static constexpr int SMEM = RING + JOIN + W * 32 * 4 + 64 * 4 + W * S * 8 + 64 + 1024;
};

struct DecodeArgs {
  const void* q;
  void* out;
  const int32_t* tables;
  const int32_t* lens;
  float* part;      // [2 * grid][16][DP] sums, then [2 * grid][16][2] (max, sum)
  uint32_t* count;  // [grid]
  int64_t q_row, q_head, o_row, o_head, table_row;
  int64_t room;     // tokens a table row has room for
  int batch, hkv, group, hblocks, d, page_size, num_pages, window;
  int one_box;      // a box holds all column blocks of its rows
  float s2;         // scale * log2(e)
};

// A walk over the blocks [u, end) of the work list: where the current item's blocks lie.
struct Walk {
  int64_t u, end, base;  // next block, end of the run, first block of the current sequence
  int b, nb, f, len, lo; // sequence: index, blocks per item, first block's index, length, first visible token
  int item, k0, n;       // current segment: item within the sequence, its first block and their number
  bool starts, ends;     // whether the segment holds the item's first / last block
};

__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b, bool* cut) {
  const int64_t l = a.lens[b];
  *cut = l > a.room;
  return static_cast<int>(l > a.room ? a.room : l < 0 ? 0 : l);
}

template <int BLOCK>
__device__ __forceinline__ int seq_blocks(const DecodeArgs& a, int len, int* lo) {
  *lo = a.window > 0 && len > a.window ? len - a.window : 0;
  return len > 0 ? (len + BLOCK - 1) / BLOCK - *lo / BLOCK : 0;
}

template <int BLOCK>
__device__ __forceinline__ void walk_load(const DecodeArgs& a, Walk& w) {
  bool cut;
  w.len = seq_len(a, w.b, &cut);
  w.nb = seq_blocks<BLOCK>(a, w.len, &w.lo);
  w.f = w.lo / BLOCK;
}

// The next segment of the run; false at its end.
template <int BLOCK>
__device__ __forceinline__ bool walk_next(const DecodeArgs& a, Walk& w, int hi) {
  if (w.u >= w.end) return false;
  while (w.nb == 0 || w.u >= w.base + static_cast<int64_t>(w.nb) * hi) {
    w.base += static_cast<int64_t>(w.nb) * hi;
    if (++w.b >= a.batch) {  // only if the lengths changed under the kernel
      w.u = w.end;
      return false;
    }
    walk_load<BLOCK>(a, w);
  }
  const int64_t off = w.u - w.base;
  w.item = static_cast<int>(off / w.nb);
  w.k0 = static_cast<int>(off - static_cast<int64_t>(w.item) * w.nb);
  w.n = static_cast<int>(min(static_cast<int64_t>(w.nb - w.k0), w.end - w.u));
  w.starts = w.k0 == 0;
  w.ends = w.k0 + w.n == w.nb;
  w.u += w.n;
  return true;
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4,
                                            uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// R: rows of a TMA box, 16, or 8 where the page size is an odd multiple of 8.
template <int DP, int DT, int R>
__global__ void __launch_bounds__(Shape<DP>::W * 32, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const __grid_constant__ DecodeArgs a) {
  using C = Shape<DP>;
  constexpr int W = C::W, S = C::S, NB = C::NB, BLOCK = C::BLOCK, T = W * 32;
  // row r, column block c of a 16-token half: (r / 8) * HS + c * BS + (r % 8) * 128
  constexpr int HS = R == 16 ? 1024 : NB * 1024, BS = R == 16 ? 2048 : 1024;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  float* join = reinterpret_cast<float*>(ring + C::RING);
  float* ml = join + C::JOIN / 4;      // [W][16][2]: each warp's max and sum per row
  float* misc = ml + W * 32;           // [64]: scan scratch
  uint64_t* bars = reinterpret_cast<uint64_t*>(misc + 64);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = bars + warp * S;
  uint8_t* mine = ring + warp * S * C::STAGE;
  if (tid == 0)
    for (int i = 0; i < W * S; ++i) mbar_init(bars + i, 1);
  fence_mbar_init();
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's run of blocks ----------------------------------------------------
  const int hi = a.hkv * a.hblocks;  // items per sequence
  int64_t* scan = reinterpret_cast<int64_t*>(misc);  // [W + 2]
  int64_t total = 0;
  {
    int64_t s = 0;
    for (int b = tid; b < a.batch; b += T) {
      int lo;
      bool cut;
      const int len = seq_len(a, b, &cut);
      if (cut && blockIdx.x == 0) atomicOr(&g_device_error, kErrIndex);
      s += seq_blocks<BLOCK>(a, len, &lo);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) scan[warp] = s;
    if (tid == 0) scan[W] = scan[W + 1] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) total += scan[i];
  }
  const int64_t blocks = total * hi;
  const int64_t runs = min(static_cast<int64_t>(gridDim.x), blocks);
  const int64_t me = blockIdx.x;
  auto run_begin = [&](int64_t c) { return c * blocks / runs; };
  Walk cw;
  cw.u = me < runs ? run_begin(me) : 0;
  cw.end = me < runs ? run_begin(me + 1) : 0;
  cw.b = 0;
  cw.base = 0;
  cw.nb = 0;
  if (cw.u < cw.end) {
    // the sequence of the run's first block: sums of blocks over tiles of T sequences
    int64_t before = 0;
    for (int b0 = 0;; b0 += T) {
      int lo, nb = 0;
      bool cut;
      if (b0 + tid < a.batch) nb = seq_blocks<BLOCK>(a, seq_len(a, b0 + tid, &cut), &lo);
      int64_t inc = nb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      __syncthreads();  // the last reads of scan
      if (lane == 31) scan[warp] = inc;
      __syncthreads();
      int64_t tile = 0, front = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (i < warp) front += scan[i];
        tile += scan[i];
      }
      const int64_t first = before + front + inc - nb;  // blocks per item before this thread's sequence
      if (nb > 0 && cw.u >= first * hi && cw.u < (first + nb) * hi) {
        scan[W] = b0 + tid;
        scan[W + 1] = first * hi;
      }
      const bool here = cw.u < (before + tile) * hi;
      before += tile;
      if (here || b0 + T >= a.batch) break;  // the total says that it is found by the last tile
    }
    __syncthreads();
    cw.b = static_cast<int>(scan[W]);
    cw.base = scan[W + 1];
    walk_load<BLOCK>(a, cw);
  }
  // sequences that see nothing: zeros
  for (int b = static_cast<int>(me); b < a.batch; b += gridDim.x) {
    int lo;
    bool cut;
    if (seq_blocks<BLOCK>(a, seq_len(a, b, &cut), &lo)) continue;
    const int per = a.d / 8, heads = a.hkv * a.group;
    for (int i = tid; i < heads * per; i += T)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + b * a.o_row + i / per * a.o_head + i % per * 8) =
          make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (cw.u >= cw.end) return;

  // ---- the producer half of each warp: the chunks of its walk, S stages ahead ---------
  Walk pw = cw;
  int pk = 0, pn = 0, pbase = 0;  // next block of the segment, their number, block of pid's lane 0
  int pid0 = 0, pid1 = 0;         // lane i: pages of the chunk's first (and second) 8 tokens, block pbase + i
  int stage_p = 0;
  bool alive = true;              // no wait has run out
  const uint64_t policy = l2_evict_first_policy();
  auto load_pages = [&]() {
    pbase = pk;
    const int t = (pw.f + pw.k0 + pk + lane) * BLOCK + warp * 16;
    const int32_t* row = a.tables + pw.b * a.table_row;
    auto page_of = [&](int tok) {
      if (tok >= pw.len || tok + R <= pw.lo) return a.num_pages;
      const int p = row[tok / a.page_size];
      if (p >= 0 && p < a.num_pages) return p;
      atomicOr(&g_device_error, kErrIndex);
      return a.num_pages;  // outside the map: the box is filled with zeros
    };
    if (pk + lane < pn) {
      pid0 = page_of(t);
      pid1 = R == 8 ? page_of(t + 8) : 0;
    }
  };
  auto produce = [&]() {  // the next chunk of this warp into its next stage, if there is one
    for (;;) {
      if (pk >= pn) {
        if (!walk_next<BLOCK>(a, pw, hi)) return;
        pk = 0;
        pn = pw.n;
        load_pages();
      } else if (pk - pbase == 32) {
        load_pages();
      }
      const int t = (pw.f + pw.k0 + pk) * BLOCK + warp * 16;
      const int sel = pk - pbase;
      ++pk;
      if (t >= pw.len || t + 16 <= pw.lo) continue;
      const int p0 = __shfl_sync(0xFFFFFFFFu, pid0, sel), p1 = __shfl_sync(0xFFFFFFFFu, pid1, sel);
      if (lane == 0) {
        uint8_t* dst = mine + stage_p * C::STAGE;
        uint64_t* bar = full + stage_p;
        const int head = pw.item / a.hblocks;
        mbar_arrive_expect_tx(bar, C::STAGE);
#pragma unroll
        for (int h = 0; h < 16 / R; ++h) {
          const int slot = (t + 8 * h) % a.page_size, page = h ? p1 : p0;
          if (a.one_box) {
            tma_load_5d(dst + h * HS, &kmap, 0, slot, 0, head, page, bar, policy);
            tma_load_5d(dst + C::HALF + h * HS, &vmap, 0, slot, 0, head, page, bar, policy);
          } else {
#pragma unroll
            for (int c = 0; c < NB; ++c) {
              tma_load_5d(dst + h * HS + c * BS, &kmap, c * 64, slot, 0, head, page, bar, policy);
              tma_load_5d(dst + C::HALF + h * HS + c * BS, &vmap, c * 64, slot, 0, head, page, bar, policy);
            }
          }
        }
      }
      stage_p = stage_p + 1 == S ? 0 : stage_p + 1;
      return;
    }
  };
#pragma unroll 1
  for (int i = 0; i < S; ++i) produce();

  // ---- the consumer half -------------------------------------------------------------
  const int g = lane >> 2, t4 = lane & 3;
  int stage_c = 0;
  uint32_t phase = 0;
  const uint32_t mine_u = smem_u32(mine);
  // ldmatrix row addresses inside a 16-token half; lane l supplies row l % 16 of an x4
  const int lr = lane & 7, lq = lane >> 3;
  while (walk_next<BLOCK>(a, cw, hi)) {
    const int head = cw.item / a.hblocks, hb = cw.item % a.hblocks;
    const int rows = min(a.group - hb * 16, 16);
    const int qh0 = head * a.group + hb * 16;
    uint32_t qf[DP / 16][4];
    {
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + cw.b * a.q_row + qh0 * a.q_head;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = g + (i & 1) * 8, c = k * 16 + t4 * 2 + (i >> 1) * 8;
          qf[k][i] = r < rows && c < a.d ? *reinterpret_cast<const uint32_t*>(qp + r * a.q_head + c) : 0u;
        }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll 1
    for (int k = 0; k < cw.n; ++k) {
      const int t = (cw.f + cw.k0 + k) * BLOCK + warp * 16;
      if (t >= cw.len || t + 16 <= cw.lo) continue;
      const uint32_t kb = mine_u + stage_c * C::STAGE, vb = kb + C::HALF;
      if (alive) alive = mbar_wait(full + stage_c, phase);
      alive = __all_sync(0xFFFFFFFFu, alive);
      if (alive) {
        const bool edge = t < cw.lo || t + 16 > cw.len;
        if (edge) {  // values past the end may be anything, NaN too: a weight of 0 must meet 0
          for (int r = max(0, cw.len - t); r < 16; ++r)
            for (int c = lane; c < NB * 8; c += 32)
              *reinterpret_cast<uint4*>(mine + stage_c * C::STAGE + C::HALF + (r >> 3) * HS + (c >> 3) * BS + (r & 7) * 128 +
                                        (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          for (int r = 0; r < min(16, cw.lo - t); ++r)
            for (int c = lane; c < NB * 8; c += 32)
              *reinterpret_cast<uint4*>(mine + stage_c * C::STAGE + C::HALF + (r >> 3) * HS + (c >> 3) * BS + (r & 7) * 128 +
                                        (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into this stage
        }
        // scores: 16 query heads x 16 tokens
        float s[2][4] = {};
#pragma unroll
        for (int k16 = 0; k16 < DP / 16; ++k16) {
          // matrices: tokens 0-7 / 8-15 x columns k16*16 + 0-7 / 8-15
          const int c = k16 * 2 + (lq & 1), cc = c & 7;
          uint32_t b[4];
          ldsm4(kb + (lq >> 1) * HS + (c >> 3) * BS + lr * 128 + ((cc ^ lr) << 4), b);
          mma_16816<DT>(s[0], qf[k16], b[0], b[1]);
          mma_16816<DT>(s[1], qf[k16], b[2], b[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][i] *= a.s2;
            const int tok = t + n * 8 + t4 * 2 + (i & 1);
            if (edge && (tok < cw.lo || tok >= cw.len)) s[n][i] = -INFINITY;
          }
        float n0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        float n1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        n0 = fmaxf(n0, __shfl_xor_sync(0xFFFFFFFFu, n0, 1));
        n1 = fmaxf(n1, __shfl_xor_sync(0xFFFFFFFFu, n1, 1));
        n0 = fmaxf(n0, __shfl_xor_sync(0xFFFFFFFFu, n0, 2));
        n1 = fmaxf(n1, __shfl_xor_sync(0xFFFFFFFFu, n1, 2));
        if (__any_sync(0xFFFFFFFFu, n0 > m0 || n1 > m1)) {
          n0 = fmaxf(n0, m0);
          n1 = fmaxf(n1, m1);
          const float f0 = exp2_fast(m0 - (n0 == -INFINITY ? 0.f : n0));
          const float f1 = exp2_fast(m1 - (n1 == -INFINITY ? 0.f : n1));
          m0 = n0;
          m1 = n1;
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][0] *= f0;
            o[i][1] *= f0;
            o[i][2] *= f1;
            o[i][3] *= f1;
          }
        }
        const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n][0] = exp2_fast(s[n][0] - z0);
          s[n][1] = exp2_fast(s[n][1] - z0);
          s[n][2] = exp2_fast(s[n][2] - z1);
          s[n][3] = exp2_fast(s[n][3] - z1);
          l0 += s[n][0] + s[n][1];
          l1 += s[n][2] + s[n][3];
        }
        // the weights, in [0, 1], rounded to the cache's type for the product with v: a
        // relative 2^-9 (2^-12) each, below the rounding of the output; their sum is not rounded
        const uint32_t p[4] = {pack16<DT>(s[0][0], s[0][1]), pack16<DT>(s[0][2], s[0][3]), pack16<DT>(s[1][0], s[1][1]),
                               pack16<DT>(s[1][2], s[1][3])};
#pragma unroll
        for (int n16 = 0; n16 < DP / 16; ++n16) {
          // matrices: tokens 0-7 / 8-15 x columns n16*16 + 0-7, then columns + 8
          const int c = n16 * 2 + (lq >> 1), cc = c & 7;
          uint32_t b[4];
          ldsm4_t(vb + (lq & 1) * HS + (c >> 3) * BS + lr * 128 + ((cc ^ lr) << 4), b);
          mma_16816<DT>(o[n16 * 2], p, b[0], b[1]);
          mma_16816<DT>(o[n16 * 2 + 1], p, b[2], b[3]);
        }
      }
      __syncwarp();
      stage_c = stage_c + 1 == S ? 0 : stage_c + 1;
      if (stage_c == 0) phase ^= 1;
      if (alive) produce();
    }
    // ---- join the warps --------------------------------------------------------------
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);
    if (t4 == 0) {
      ml[(warp * 16 + g) * 2] = m0;
      ml[(warp * 16 + g) * 2 + 1] = l0;
      ml[(warp * 16 + g + 8) * 2] = m1;
      ml[(warp * 16 + g + 8) * 2 + 1] = l1;
    }
    __syncthreads();
    const bool whole = cw.starts && cw.ends;
    const int64_t seg0 = cw.u - cw.n;                               // first block of the segment
    const int64_t item0 = cw.base + static_cast<int64_t>(cw.item) * cw.nb;  // first block of the item
    const int slot = static_cast<int>(me) * 2 + (seg0 == run_begin(me) ? 0 : 1);
    float* part_o = a.part + static_cast<int64_t>(slot) * 16 * DP;
    float* part_ml = a.part + static_cast<int64_t>(2 * gridDim.x) * 16 * DP + slot * 32;
    uint16_t* outp = static_cast<uint16_t*>(a.out) + cw.b * a.o_row + qh0 * a.o_head;
#pragma unroll 1
    for (int h = 0; h * 8 < rows; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mx = fmaxf(mx, ml[(w * 16 + h * 8 + g) * 2]);
      const float z = mx == -INFINITY ? 0.f : mx;
      const float f = exp2_fast((h ? m1 : m0) - z);
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const float x = h ? o[i][2] : o[i][0], y = h ? o[i][3] : o[i][1];
        *reinterpret_cast<float2*>(join + (warp * 8 + g) * DP + i * 8 + t4 * 2) = make_float2(x * f, y * f);
      }
      __syncthreads();
      for (int e = tid; e < 8 * DP / 4; e += T) {
        const int r = e / (DP / 4), c = e % (DP / 4) * 4, row = h * 8 + r;
        if (row >= rows) continue;
        float mr = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) mr = fmaxf(mr, ml[(w * 16 + row) * 2]);
        const float zr = mr == -INFINITY ? 0.f : mr;
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          l += ml[(w * 16 + row) * 2 + 1] * exp2_fast(ml[(w * 16 + row) * 2] - zr);
          const float4 v = *reinterpret_cast<const float4*>(join + (w * 8 + r) * DP + c);
          acc.x += v.x;
          acc.y += v.y;
          acc.z += v.z;
          acc.w += v.w;
        }
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          if (c < a.d)
            *reinterpret_cast<uint2*>(outp + row * a.o_head + c) =
                make_uint2(pack16<DT>(acc.x * inv, acc.y * inv), pack16<DT>(acc.z * inv, acc.w * inv));
        } else {
          __stcg(reinterpret_cast<float4*>(part_o + row * DP + c), acc);
          if (c == 0) __stcg(reinterpret_cast<float2*>(part_ml + row * 2), make_float2(mr, l));
        }
      }
      __syncthreads();
    }
    if (whole) continue;
    // ---- join the CTAs of this item: the last one to arrive adds the partials ----------
    auto run_of = [&](int64_t block) {  // the run that holds a block
      int64_t c = block * runs / blocks;
      while (run_begin(c + 1) <= block) ++c;
      while (run_begin(c) > block) --c;
      return c;
    };
    const int64_t c0 = run_of(item0), c1 = run_of(item0 + cw.nb - 1);
    if (tid == 0) {
      __threadfence();
      misc[63] = __uint_as_float(atomicAdd(a.count + c0, 1u));
      __threadfence();
    }
    __syncthreads();
    if (__float_as_uint(misc[63]) + 1 != static_cast<uint32_t>(c1 - c0 + 1)) continue;
    if (tid == 0) a.count[c0] = 0;
    const int slot0 = static_cast<int>(c0) * 2 + (item0 == run_begin(c0) ? 0 : 1);
    const float* po = a.part;
    const float* pm = a.part + static_cast<int64_t>(2 * gridDim.x) * 16 * DP;
    for (int e = tid; e < rows * (DP / 4); e += T) {
      const int row = e / (DP / 4), c = e % (DP / 4) * 4;
      float mr = -INFINITY;
      for (int64_t k = c0; k <= c1; ++k) {
        const int64_t sl = k == c0 ? slot0 : 2 * k;
        mr = fmaxf(mr, __ldcg(pm + sl * 32 + row * 2));
      }
      const float zr = mr == -INFINITY ? 0.f : mr;
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int64_t k = c0; k <= c1; ++k) {
        const int64_t sl = k == c0 ? slot0 : 2 * k;
        const float2 mk = __ldcg(reinterpret_cast<const float2*>(pm + sl * 32 + row * 2));
        const float4 v = __ldcg(reinterpret_cast<const float4*>(po + (sl * 16 + row) * DP + c));
        const float f = exp2_fast(mk.x - zr);
        l += mk.y * f;
        acc.x += v.x * f;
        acc.y += v.y * f;
        acc.z += v.z * f;
        acc.w += v.w * f;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (c < a.d)
        *reinterpret_cast<uint2*>(outp + row * a.o_head + c) =
            make_uint2(pack16<DT>(acc.x * inv, acc.y * inv), pack16<DT>(acc.z * inv, acc.w * inv));
    }
  }
  // every copy this warp issued was waited for unless a wait ran out: those left, with a limit
  if (!alive)
    for (int i = 0; i < S; ++i) {
      mbar_wait(full + stage_c, phase);
      stage_c = stage_c + 1 == S ? 0 : stage_c + 1;
      if (stage_c == 0) phase ^= 1;
    }
}

// The cache as [pages][heads][column blocks][slots][64], or, where the head is no multiple
// of 64 wide, [pages][heads][1][slots][d] with boxes that reach past d (filled with zeros).
bool make_cache_map(CUtensorMap* map, const void* base, int64_t dtype, const ggufmm_attention_args& p, int64_t page,
                    int64_t head, int64_t slot, int rows, bool one_box) {
  PFN_encodeTiled enc = get_encode_fn();
  if (!enc) return false;
  const cuuint64_t d = static_cast<cuuint64_t>(p.head_dim), cols = one_box ? d / 64 : 1;
  cuuint64_t dims[5] = {one_box ? 64 : d, static_cast<cuuint64_t>(p.page_size), cols,
                        static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.num_pages)};
  cuuint64_t strides[4] = {static_cast<cuuint64_t>(slot) * 2, 128, static_cast<cuuint64_t>(head) * 2,
                           static_cast<cuuint64_t>(page) * 2};
  cuuint32_t box[5] = {64, static_cast<cuuint32_t>(rows), static_cast<cuuint32_t>(cols), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(map, dtype == GGUFMM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int DT, int R>
cudaError_t launch(const ggufmm_attention_args& p, DecodeArgs& a, int grid, int dev, cudaStream_t st) {
  CUtensorMap km, vm;
  if (!make_cache_map(&km, p.k, p.dtype, p, p.k_page, p.k_head, p.k_slot, R, a.one_box) ||
      !make_cache_map(&vm, p.v, p.dtype, p, p.v_page, p.v_head, p.v_slot, R, a.one_box))
    return cudaErrorInvalidValue;
  auto fn = paged_decode_kernel<DP, DT, R>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  if (!(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::SMEM);
    if (e != cudaSuccess) return e;
    ready.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_release);
  }
  return pdl_launch(fn, dim3(static_cast<unsigned>(grid)), dim3(Shape<DP>::W * 32), Shape<DP>::SMEM, st, km, vm, a);
}

template <int DP>
cudaError_t launch_dp(const ggufmm_attention_args& p, DecodeArgs& a, int grid, int dev, cudaStream_t st) {
  const bool f16 = p.dtype == GGUFMM_F16;
  if (p.page_size % 16 == 0)
    return f16 ? launch<DP, GGUFMM_F16, 16>(p, a, grid, dev, st) : launch<DP, GGUFMM_BF16, 16>(p, a, grid, dev, st);
  return f16 ? launch<DP, GGUFMM_F16, 8>(p, a, grid, dev, st) : launch<DP, GGUFMM_BF16, 8>(p, a, grid, dev, st);
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

}  // namespace

size_t paged_decode_workspace(int64_t head_dim) {
  return kCounterBytes + static_cast<size_t>(2 * kMaxGrid) * 16 * (padded_dim(head_dim) + 2) * 4;
}

cudaError_t launch_paged_decode(const ggufmm_attention_args& p, void* workspace, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int grid = std::min(std::max(device_info(dev).sms, 1), kMaxGrid);
  DecodeArgs a;
  a.q = p.q;
  a.out = p.out;
  a.tables = static_cast<const int32_t*>(p.tables);
  a.lens = static_cast<const int32_t*>(p.lens);
  a.count = static_cast<uint32_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  a.q_row = p.q_row;
  a.q_head = p.q_head;
  a.o_row = p.o_row;
  a.o_head = p.o_head;
  a.table_row = p.table_row;
  a.room = p.table_width * p.page_size;
  a.batch = static_cast<int>(p.batch);
  a.hkv = static_cast<int>(p.kv_heads);
  a.group = static_cast<int>(p.q_heads / p.kv_heads);
  a.hblocks = (a.group + 15) / 16;
  a.d = static_cast<int>(p.head_dim);
  a.page_size = static_cast<int>(p.page_size);
  a.num_pages = static_cast<int>(p.num_pages);
  a.window = static_cast<int>(p.window);
  a.one_box = a.d % 64 == 0 && a.d == padded_dim(a.d);
  a.s2 = static_cast<float>(p.scale * 1.4426950408889634);
  switch (padded_dim(p.head_dim)) {
    case 64: return launch_dp<64>(p, a, grid, dev, st);
    case 128: return launch_dp<128>(p, a, grid, dev, st);
    default: return launch_dp<256>(p, a, grid, dev, st);
  }
}

cudaError_t attn_decode_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }
cudaError_t attn_decode_set_wait_limit(uint32_t polls) { return tu_set_wait_limit(polls); }

}  // namespace ggufmm
