// attn_prompt.cu -- ggufmm_paged_prompt_attention: causal attention of ragged runs of new
// tokens over the paged key-value cache, on the tcgen05 tensor cores.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_j p_ij,  p_ij = 2^(s_ij - m_i),  s_ij = scale log2(e) q_i.k_j
//
// One pass over the keys with a running maximum m_i and sum; scores and weights stay in
// tensor memory and registers. The work is 4 D flops per (query head, key) pair at length,
// tensor bound, with one exponential per pair next to it: a special-function unit makes 16
// a clock per SM, the tensor cores 128 x 128 pairs of D = 128 in about 1024 clocks, so the
// two are nearly equal and have to overlap.
//
// Tiles: the G query heads of a kv head and floor(128 / G) consecutive tokens are the 128
// rows of one query tile (row = token * G + head), so short prompts fill tiles and every key
// is loaded once for the whole group. A CTA holds two query tiles (one for heads wider than
// 128): while the softmax warps of one work on its scores, the tensor core multiplies for the
// other. Keys and values come page by page by TMA into 128-row (64-row) swizzled tiles; q k^T
// goes to TMEM, thread r of a softmax warpgroup reads row r, writes the weights back over the
// scores as 16-bit values, and the second product reads them from TMEM. The running output
// stays in TMEM; it is rescaled only when a row's maximum has grown by more than 2^8 since its
// last rescaling (the weights then reach at most 2^8, harmless in 32-bit sums).
//
// Warps: 4 softmax warps per query tile, one that loads, one that issues the products.
#include <algorithm>
#include <atomic>

#include "mma16.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace ggufmm {

namespace {

template <int DP>
struct PShape {
  static constexpr int NQ = DP == 256 ? 1 : 2;     // query tiles
  static constexpr int BN = DP == 256 ? 64 : 128;  // keys of a tile
  static constexpr int NB = DP / 64;               // 128-byte column blocks of a row
  static constexpr int NS = 2;                     // score buffers: one per query tile, or two in turn
  static constexpr int KS = 2, VS = 2;             // stages
  static constexpr int QB = 128 * DP * 2, KB = BN * DP * 2;
  static constexpr int BARS = NQ * QB + (KS + VS) * KB;
  static constexpr int SMEM = BARS + 256 + 1024;
  static constexpr int SCOL = BN;                  // TMEM columns of a score buffer
  static constexpr int OCOL = NS * BN;             // first column of the outputs
  static constexpr int COLS = OCOL + NQ * DP <= 256 ? 256 : 512;
  static constexpr int THREADS = NQ * 128 + 64;
};

struct PromptArgs {
  void* out;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* starts;
  int64_t o_row, o_head, table_row, room, total_q;
  int batch, hkv, group, toks, tiles, d, page_size, num_pages, window, max_q;
  int box;   // rows of a K / V box
  float s2;  // scale * log2(e)
};

// A [tokens][64 columns] block of 128-byte rows read with the columns as the long (N)
// dimension: 64-column blocks `block` bytes apart, groups of 8 tokens 1024 apart.
__device__ __forceinline__ uint64_t umma_smem_desc_mn(uint32_t saddr, uint32_t block) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <int DT, int N, bool BMN>
__device__ __forceinline__ constexpr uint32_t idesc16() {
  constexpr uint32_t ty = DT == GGUFMM_BF16 ? 1u : 0u;
  return (1u << 4) | (ty << 7) | (ty << 10) | (BMN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (8u << 24);
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  umma_f16(d, a, b, idesc, acc ? 1u : 0u);
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc ? 1u : 0u)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t));
}
__device__ __forceinline__ void tmem_st32(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31]), "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}

template <int DP, int DT>
__global__ void __launch_bounds__(PShape<DP>::THREADS, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PromptArgs a) {
  using C = PShape<DP>;
  constexpr int NQ = C::NQ, BN = C::BN, NB = C::NB, KS = C::KS, VS = C::VS;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sk = sq + NQ * C::QB;
  uint8_t* sv = sk + KS * C::KB;
  uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + C::BARS);
  uint64_t* kfull = qfull + 1;
  uint64_t* kempty = kfull + KS;
  uint64_t* vfull = kempty + KS;
  uint64_t* vempty = vfull + VS;
  uint64_t* vfix = vempty + VS;
  uint64_t* sfull = vfix + 1;   // [2] scores in a buffer
  uint64_t* pready = sfull + 2; // [2] weights in a buffer
  uint64_t* odone = pready + 2; // [2] a query tile's product with the values is done
  uint32_t* slot = reinterpret_cast<uint32_t*>(odone + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();

  // ---- what this CTA works on: heads fastest, the longest (latest) tiles first -----------
  const int per = a.hkv * a.batch;
  const int tile = a.tiles - 1 - static_cast<int>(blockIdx.x) / per;
  const int bh = static_cast<int>(blockIdx.x) % per, b = bh / a.hkv, head = bh % a.hkv;
  const int q0 = a.starts[b], n_all = a.starts[b + 1] - q0;
  const int n = q0 < 0 || q0 > a.total_q ? 0 : static_cast<int>(min(static_cast<int64_t>(min(n_all, a.max_q)), a.total_q - q0));
  const int64_t len64 = a.lens[b];
  const int len = static_cast<int>(len64 < 0 ? 0 : len64 > a.room ? a.room : len64);
  if (tile == 0 && head == 0 && threadIdx.x == 0 && (n < n_all || n_all < 0 || len < len64))
    atomicOr(&g_device_error, kErrIndex);
  const int t0 = tile * NQ * a.toks;  // first token of the CTA
  if (t0 >= n) return;
  const int first = len - n_all + t0;                                    // its position
  const int end = len - n_all + min(n, t0 + NQ * a.toks);                 // one past the last query's
  const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int j0 = lo / BN;
  const int nt = end > 0 ? (end + BN - 1) / BN - j0 : 0;  // key tiles

  uint16_t* outp = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(head) * a.group * a.o_head;
  if (nt <= 0) {  // every query lies before position 0
    const int c8 = a.d / 8, cnt = min(NQ * a.toks, n - t0) * a.group * c8;
    for (int i = threadIdx.x; i < cnt; i += C::THREADS) {
      const int c = i % c8, g = i / c8 % a.group, t = i / c8 / a.group;
      *reinterpret_cast<uint4*>(outp + static_cast<int64_t>(q0 + t0 + t) * a.o_row + g * a.o_head + c * 8) =
          make_uint4(0, 0, 0, 0);
    }
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(qfull, 1);
    for (int i = 0; i < KS; ++i) mbar_init(kfull + i, 1), mbar_init(kempty + i, 1);
    for (int i = 0; i < VS; ++i) mbar_init(vfull + i, 1), mbar_init(vempty + i, 1);
    mbar_init(vfix, 1);
    for (int i = 0; i < 2; ++i) mbar_init(sfull + i, 1), mbar_init(pready + i, 4), mbar_init(odone + i, 1);
    fence_mbar_init();
  }
  if (warp == NQ * 4 + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(static_cast<uint32_t>(C::COLS))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *slot;
  // not earlier: a dependent kernel that takes its tensor memory before it waits for this
  // grid must find that all of this grid's CTAs have theirs
  pdl_trigger();

  if (warp == NQ * 4) {
    // ---- loads -------------------------------------------------------------------------
    bool ok = true;
    int kt = 0, vt = 0;  // tiles asked for
    if (lane == 0) mbar_arrive_expect_tx(qfull, NQ * NB * a.toks * a.group * 128);
    __syncwarp();
    if (lane < NQ * NB) {
      const int i = lane / NB, c = lane % NB;
      tma_load_4d(sq + i * C::QB + c * (128 * 128), &qmap, c * 64, 0, head, q0 + t0 + i * a.toks, qfull);
    }
    const int32_t* row = a.tables + b * a.table_row;
    const int boxes = NB * (BN / a.box);
    auto load = [&](uint8_t* dst, const CUtensorMap* map, int j, uint64_t* bar) {
      if (lane == 0) mbar_arrive_expect_tx(bar, C::KB);
      __syncwarp();
      for (int x = lane; x < boxes; x += 32) {
        const int c = x % NB, r = x / NB * a.box, tok = j * BN + r;
        int page = a.num_pages;  // outside the map: the box is filled with zeros
        if (tok < len && tok + a.box > lo) {
          const int p = row[tok / a.page_size];
          if (p >= 0 && p < a.num_pages) page = p;
          else atomicOr(&g_device_error, kErrIndex);
        }
        tma_load_4d(dst + c * (BN * 128) + r * 128, map, c * 64, tok % a.page_size, head, page, bar);
      }
    };
    for (int t = 0; t < nt && ok; ++t) {
      const int ks = t % KS, vs = t % VS, j = j0 + t;
      ok = mbar_wait(kempty + ks, (t / KS & 1) ^ 1);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      load(sk + ks * C::KB, &kmap, j, kfull + ks);
      ++kt;
      ok = mbar_wait(vempty + vs, (t / VS & 1) ^ 1);
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
      // tokens past the length that share a box with some before it may hold anything, NaN
      // too, and a weight of 0 must meet 0: that tile's values are cleared there by hand
      if ((j + 1) * BN > len && len % a.box) {
        load(sv + vs * C::KB, &vmap, j, vfix);
        ok = mbar_wait(vfix, 0);  // at most once: it is the last tile of the sequence
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
        const int r0 = len - j * BN, rows = (r0 + a.box - 1) / a.box * a.box - r0;
        for (int x = lane; x < rows * NB * 8; x += 32)
          *reinterpret_cast<uint4*>(sv + vs * C::KB + x / 8 % NB * (BN * 128) + (r0 + x / 8 / NB) * 128 + x % 8 * 16) =
              make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(vfull + vs);
      } else {
        load(sv + vs * C::KB, &vmap, j, vfull + vs);
      }
      ++vt;
    }
    if (!__all_sync(0xFFFFFFFFu, ok)) {  // a wait ran out: the copies still in flight
      mbar_wait(qfull, 0);
      for (int t = max(0, kt - KS); t < kt; ++t) mbar_wait(kfull + t % KS, t / KS & 1);
      for (int t = max(0, vt - VS); t < vt; ++t) mbar_wait(vfull + t % VS, t / VS & 1);
    }
  } else if (warp == NQ * 4 + 1) {
    // ---- products ----------------------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t id_qk = idesc16<DT, BN, false>(), id_pv = idesc16<DT, DP, true>();
      auto qk = [&](int i, int buf, int ks) {  // scores of query tile i
        const uint32_t qa = smem_u32(sq + i * C::QB), ka = smem_u32(sk + ks * C::KB);
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          const uint64_t qd = umma_smem_desc(qa + c * (128 * 128)), kd = umma_smem_desc(ka + c * (BN * 128));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_ss(tmem + buf * C::SCOL, qd + 2 * k, kd + 2 * k, id_qk, c > 0 || k > 0);
        }
        umma_commit(sfull + buf);
      };
      auto pv = [&](int i, int buf, int vs, bool acc) {
        const uint64_t vd = umma_smem_desc_mn(smem_u32(sv + vs * C::KB), BN * 128);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          umma_ts(tmem + C::OCOL + i * DP, tmem + buf * C::SCOL + 8 * k, vd + k * (2048 >> 4), id_pv, acc || k > 0);
        umma_commit(odone + i);
      };
      bool ok = mbar_wait(qfull, 0) && mbar_wait(kfull, 0);
      fence_after();
      if (ok) {
        for (int i = 0; i < NQ; ++i) qk(i, i, 0);
        umma_commit(kempty);
      }
      for (int t = 0; t < nt && ok; ++t) {
        const int vs = t % VS, kn = (t + 1) % KS;
        const bool more = t + 1 < nt;
        if (NQ == 1) {
          if (more) {  // the other score buffer: its weights were read by the last product
            ok = mbar_wait(kfull + kn, (t + 1) / KS & 1);
            if (!ok) break;
            fence_after();
            qk(0, (t + 1) & 1, kn);
            umma_commit(kempty + kn);
          }
          ok = mbar_wait(vfull + vs, t / VS & 1) && mbar_wait(pready + (t & 1), t >> 1 & 1);
          if (!ok) break;
          fence_after();
          pv(0, t & 1, vs, t > 0);
        } else {
          ok = mbar_wait(vfull + vs, t / VS & 1);
          for (int i = 0; i < NQ && ok; ++i) {
            ok = mbar_wait(pready + i, t & 1);
            if (!ok) break;
            fence_after();
            pv(i, i, vs, t > 0);
            if (more) {  // over the weights just read: products run in the order of their issue
              if (i == 0) {
                ok = mbar_wait(kfull + kn, (t + 1) / KS & 1);
                if (!ok) break;
                fence_after();
              }
              qk(i, i, kn);
            }
          }
          if (!ok) break;
          if (more) umma_commit(kempty + kn);
        }
        umma_commit(vempty + vs);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread r of a warpgroup has row r of its query tile ---------------------
    const int i = warp >> 2, r = (warp & 3) * 32 + lane;
    const int tok = t0 + i * a.toks + r / a.group, g = r % a.group;
    const bool live = r < a.toks * a.group && tok < n;
    const int pos = len - n_all + tok;  // this row's position
    const int pos_a = len - n_all + t0 + i * a.toks, pos_b = pos_a + a.toks - 1;  // the tile's first and last
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    // 16-bit floats underflow early: their weights are kept 2^7 larger (the sum too)
    constexpr float kUp = DT == GGUFMM_F16 ? 7.f : 0.f;
    const bool odd_scale = a.s2 <= 0.f;
    const float s2 = odd_scale ? 1.f : a.s2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < nt; ++t) {
      const int buf = NQ == 1 ? t & 1 : i, par = NQ == 1 ? t >> 1 & 1 : t & 1;
      ok = mbar_wait(sfull + buf, par);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      fence_after();
      uint32_t sr[BN];
      const uint32_t sc = lanes + buf * C::SCOL;
#pragma unroll
      for (int c = 0; c < BN; c += 32) tmem_ld32(sc + c, sr + c);
      tmem_wait_ld();
      float* s = reinterpret_cast<float*>(sr);
      if (odd_scale) {
#pragma unroll
        for (int c = 0; c < BN; ++c) s[c] *= a.s2;
      }
      const int jb = (j0 + t) * BN;
      if (jb + BN - 1 > pos_a || (a.window > 0 && jb <= pos_b - a.window)) {
        const int up = pos - jb, dn = a.window > 0 ? pos - a.window - jb : -1;  // visible: dn < c <= up
#pragma unroll
        for (int c = 0; c < BN; ++c)
          if (c > up || c <= dn) s[c] = -INFINITY;
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < BN; c += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[c + e]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * s2;
      // rescale when the maximum has grown by more than 8 (or is the first)
      float f = 1.f;
      if (top > m + 8.f || (m == -INFINITY && top > m)) {
        f = exp2_fast(m - top);  // 0 for the first
        m = top;
        l *= f;
      }
      if (t > 0 && __any_sync(0xFFFFFFFFu, f != 1.f)) {
        ok = mbar_wait(odone + i, (t - 1) & 1);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        fence_after();
        const uint32_t oc = lanes + C::OCOL + i * DP;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(oc + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(oc + c, o);
        }
      }
      const float z = (m == -INFINITY ? 0.f : m) - kUp;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < BN; h += 64) {
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          float e[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            e[x] = exp2_fast(fmaf(s[h + c + x], s2, -z));
            sum[x] += e[x];
          }
          // rounded to the cache's type for the product, the sum is not: a relative 2^-9
          // (2^-12) of each weight, below the rounding of the output
          p[c / 2] = pack16<DT>(e[0], e[1]);
          p[c / 2 + 1] = pack16<DT>(e[2], e[3]);
        }
        tmem_st32(sc + h / 2, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pready + buf);
    }
    if (ok) ok = mbar_wait(odone + i, (nt - 1) & 1);
    ok = __all_sync(0xFFFFFFFFu, ok);
    if (ok) {
      fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* dst = outp + static_cast<int64_t>(q0 + tok) * a.o_row + g * a.o_head;
      const uint32_t oc = lanes + C::OCOL + i * DP;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        tmem_ld32(oc + c, o);
        tmem_wait_ld();
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (c + e >= a.d) break;
            uint4 v;
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float p = l == 0.f ? 0.f : __uint_as_float(o[e + 2 * x]) * inv;
              const float q = l == 0.f ? 0.f : __uint_as_float(o[e + 2 * x + 1]) * inv;
              w[x] = pack16<DT>(p, q);
            }
            *reinterpret_cast<uint4*>(dst + c + e) = v;
          }
        }
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == NQ * 4 + 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(static_cast<uint32_t>(C::COLS))
                 : "memory");
  }
}

bool encode4(CUtensorMap* map, int64_t dtype, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
             const cuuint32_t* box) {
  PFN_encodeTiled enc = get_encode_fn();
  if (!enc) return false;
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, dtype == GGUFMM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int DT>
cudaError_t launch(const ggufmm_attention_args& p, cudaStream_t st) {
  using C = PShape<DP>;
  const cuuint64_t d = static_cast<cuuint64_t>(p.head_dim), g = static_cast<cuuint64_t>(p.q_heads / p.kv_heads);
  PromptArgs a;
  a.out = p.out;
  a.tables = static_cast<const int32_t*>(p.tables);
  a.lens = static_cast<const int32_t*>(p.lens);
  a.starts = static_cast<const int32_t*>(p.q_starts);
  a.o_row = p.o_row;
  a.o_head = p.o_head;
  a.table_row = p.table_row;
  a.room = p.table_width * p.page_size;
  a.total_q = p.total_q;
  a.batch = static_cast<int>(p.batch);
  a.hkv = static_cast<int>(p.kv_heads);
  a.group = static_cast<int>(g);
  a.toks = 128 / a.group;
  a.max_q = static_cast<int>(p.max_q);
  a.tiles = (a.max_q + C::NQ * a.toks - 1) / (C::NQ * a.toks);
  a.d = static_cast<int>(p.head_dim);
  a.page_size = static_cast<int>(p.page_size);
  a.num_pages = static_cast<int>(p.num_pages);
  a.window = static_cast<int>(p.window);
  a.s2 = static_cast<float>(p.scale * 1.4426950408889634);
  a.box = 8;  // the largest run of rows up to a tile that divides a page
  while (a.box < C::BN && p.page_size % (2 * a.box) == 0) a.box *= 2;
  const int64_t ctas = static_cast<int64_t>(a.tiles) * a.hkv * a.batch;
  if (ctas > kI32Max) return cudaErrorInvalidConfiguration;
  CUtensorMap qm, km, vm;
  const cuuint64_t qd[4] = {d, g, static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.total_q)};
  const cuuint64_t qs[3] = {static_cast<cuuint64_t>(p.q_head) * 2, static_cast<cuuint64_t>(p.q_head) * g * 2,
                            static_cast<cuuint64_t>(p.q_row) * 2};
  const cuuint32_t qb[4] = {64, static_cast<cuuint32_t>(g), 1, static_cast<cuuint32_t>(a.toks)};
  const cuuint64_t cd[4] = {d, static_cast<cuuint64_t>(p.page_size), static_cast<cuuint64_t>(p.kv_heads),
                            static_cast<cuuint64_t>(p.num_pages)};
  const cuuint64_t ks[3] = {static_cast<cuuint64_t>(p.k_slot) * 2, static_cast<cuuint64_t>(p.k_head) * 2,
                            static_cast<cuuint64_t>(p.k_page) * 2};
  const cuuint64_t vs[3] = {static_cast<cuuint64_t>(p.v_slot) * 2, static_cast<cuuint64_t>(p.v_head) * 2,
                            static_cast<cuuint64_t>(p.v_page) * 2};
  const cuuint32_t cb[4] = {64, static_cast<cuuint32_t>(a.box), 1, 1};
  if (!encode4(&qm, p.dtype, p.q, qd, qs, qb) || !encode4(&km, p.dtype, p.k, cd, ks, cb) ||
      !encode4(&vm, p.dtype, p.v, cd, vs, cb))
    return cudaErrorInvalidValue;
  auto fn = paged_prompt_kernel<DP, DT>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  if (!(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    ready.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_release);
  }
  return pdl_launch(fn, dim3(static_cast<unsigned>(ctas)), dim3(C::THREADS), C::SMEM, st, qm, km, vm, a);
}

}  // namespace

cudaError_t launch_paged_prompt(const ggufmm_attention_args& p, cudaStream_t st) {
  const bool f16 = p.dtype == GGUFMM_F16;
  if (p.head_dim <= 64) return f16 ? launch<64, GGUFMM_F16>(p, st) : launch<64, GGUFMM_BF16>(p, st);
  if (p.head_dim <= 128) return f16 ? launch<128, GGUFMM_F16>(p, st) : launch<128, GGUFMM_BF16>(p, st);
  return f16 ? launch<256, GGUFMM_F16>(p, st) : launch<256, GGUFMM_BF16>(p, st);
}

cudaError_t attn_prompt_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }
cudaError_t attn_prompt_set_wait_limit(uint32_t polls) { return tu_set_wait_limit(polls); }

}  // namespace ggufmm
