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
// 128, or where no sequence has more new tokens than one holds: 4 on 131072 take 97 us with one,
// 122 with two, 4 each of 32 on 2000 52 or 69) and walks the keys 128 (64) at a time. Keys and values come page by page into swizzled
// tiles of one ring in shared memory; q k^T goes to TMEM, thread r of a softmax warpgroup
// takes row r into registers, writes the weights to TMEM as 16-bit values, and the second
// product reads them from there. Tensor memory holds two outputs of 128 columns, two sets of
// weights of 64 and ONE score buffer of 128: it is free again as soon as a warpgroup has its
// scores in registers, so the two query tiles take turns with it, each tile's next scores are
// there when its softmax has done with the last ones, and the products run in between.
// Measured for 8192 tokens of 32 / 8 heads of 128 on the way: weights written over the scores
// (so that scores, softmax and output of a tile take turns) 495 us, 64-key tiles with two
// score buffers per query tile 490 us (a product of 64 columns takes as long as one of 128).
// The running output stays in TMEM; it is rescaled only when a row's maximum has grown by more
// than 2^8 since its last rescaling (the weights then reach at most 2^8, harmless in 32-bit
// sums).
//
// A CTA stays and takes one unit of work (a pair of query tiles) after another: when the loads of
// one are under way its loading warp asks the hardware for a unit that no CTA has begun, so that
// the loads and first scores of the next run under the last softmax and the output of this one.
// One CTA per unit, or this: 2048 tokens 40.9 or 38.5 us, 8 prompts of 512 47 or 36, 32 of 128 38 or
// 28, 8192 with a window of 1024 190 or 142; one short prompt, where a CTA has one unit, 0.3 us more.
// Units are those of the sequences' own lengths, found on the device: 2048 new tokens beside 63
// single ones take 112 us, 235 with units for the longest in every sequence.
//
// 8192 tokens of 32 / 8 heads of 128: called on end, under the power limit, 491 us, 1120 TFLOP/s, 79%
// of the sustained bf16 rate; in short bursts 421 us, 1307 TFLOP/s, 79% of the burst rate. 4096 tokens,
// heads of 64, 80, 96, 128, 192, 256: 104, 112, 112, 118, 268, 252 us, of floors of 41, 52, 62, 83, 124,
// 165 (widths are padded to 64, 128 or 256). Per 256 x 128
// scores the tensor core and the exponentials are each busy for about 2050 of 3100 clocks; what
// is left is each tile's chain of load, maximum, exponentials and hand-over (2500). A
// quarter of the exponentials as polynomials on the FMA units took 3% longer.
//
// Where the query tiles are fewer than the SMs and the cache may be long (a few new tokens on a
// long text), several CTAs take shares of a tile's keys, leave fp32 partials (maximum, sum,
// output) in the workspace, and a second kernel adds them in order, a warp a row. How long the
// texts are is known on the device alone, so a CTA takes at least kMinShare key tiles, and one
// that gets them all writes the output itself. 32 / 8 heads of 128, shared out or not: 64 new
// tokens on 32768 53 or 420 us, 4 on 131072 97 or 1650, 256 on 4096 32 or 56, 100 on 2000 28 or
// 33; with less than 8 tiles in truth the second launch costs 4 us of 13 for nothing.
//
// Warps: 4 softmax warps per query tile, one that loads queries and values, one that issues
// the products, two that load keys.
#include <cuda/ptx>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mma16.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace ggufmm {

namespace {

template <int DP, int QT>  // QT: query tiles of a CTA
struct PShape {
  static_assert(QT == 1 || (QT == 2 && DP < 256), "two outputs of 256 columns leave no room for scores");
  static constexpr int NQ = QT;
  static constexpr int BN = DP == 256 ? 64 : 128;  // keys of a tile
  static constexpr int NB = DP / 64;               // 128-byte column blocks of a row
  static constexpr int QB = 128 * DP * 2, KB = BN * DP * 2;
  static constexpr int SLOTS = DP == 64 ? 10 : DP == 128 && QT == 1 ? 6 : 5;  // tiles of keys or values in flight
  static constexpr int BARS = NQ * QB + SLOTS * KB;
  static constexpr int NBARS = 8 + 2 * SLOTS + 5 * NQ;
  static constexpr int PLAN = (BARS + NBARS * 8 + 15) / 16 * 16;  // Plan, a 16-byte answer, a word
  static constexpr int SMEM = PLAN + 64 + 16 + 16;
  static_assert(SMEM <= 232448, "a CTA's shared memory");
  // TMEM columns: one score buffer for all query tiles, their weights, their outputs
  static constexpr int PCOL = BN, OCOL = PCOL + NQ * BN / 2, COLS = 512;
  static_assert(OCOL + NQ * DP <= COLS, "tensor memory");
  static constexpr int OW = NQ * 4;                // first of the other warps
  static constexpr int THREADS = NQ * 128 + 128;
};

constexpr int kMinShare = 8;      // key tiles of a CTA where the keys are shared out
constexpr int kLaunchRegs = 168;  // a thread's at launch, where warps shift registers: (208 + 208 + 88) / 3

struct PromptArgs {
  void* out;
  const uint16_t* k;
  int64_t k_page, k_head, k_slot;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* starts;
  int64_t o_row, o_head, table_row, room, total_q;
  float* part;  // splits > 1: [units][splits][rows][DP] outputs, then [units][splits][rows][2] (max, sum)
  int batch, hkv, group, toks, tiles, d, page_size, num_pages, window, max_q, splits, units;
  int box;      // rows of a K / V box
  int one_box;  // a V box holds all column blocks of its rows
  float s2;  // scale * log2(e)
  uint32_t polls;  // of the wait for another unit before it gives up, 0: mbar_wait's limit
};

// One unit of work: a pair (one) of query tiles of a sequence and kv head.
struct Unit {
  int b, head, q0, n, base, len;  // n: new tokens that there is room for; base: position of the first
  int t0, lo;                     // first token, first visible position
  int all, share;                 // key tiles, and those of a CTA
};

// The new tokens from q0 on that there is room for, of the n that the caller gives a sequence.
__device__ __forceinline__ int new_tokens(const PromptArgs& a, int q0, int n) {
  const int room = q0 < 0 || q0 > a.total_q ? 0 : static_cast<int>(min(static_cast<int64_t>(a.max_q), a.total_q - q0));
  return max(min(n, room), 0);
}

// Unit x, by a warp: heads fastest, then the sequences that have a tile as late as this one, the
// latest tiles (the longest) first. Sequences with few new tokens beside others with many take no
// more units than they have tiles. False past the last one.
template <int DP, int QT>
__device__ __forceinline__ bool unit_of(const PromptArgs& a, int x, Unit& u) {
  using C = PShape<DP, QT>;
  const int lane = threadIdx.x & 31, per = C::NQ * a.toks;
  auto tiles_of = [&](int b) {
    if (b >= a.batch) return 0;
    const int q0 = a.starts[b];
    return (new_tokens(a, q0, a.starts[b + 1] - q0) + per - 1) / per;
  };
  // the first 32 sequences stay in registers: one wait for memory, not three
  const bool there = lane < a.batch;
  const int start = there ? a.starts[lane] : 0, given = there ? a.starts[lane + 1] - start : 0, held = there ? a.lens[lane] : 0;
  const int first = (new_tokens(a, start, given) + per - 1) / per;
  auto count = [&](int tile) {  // of tiles from `tile` on, of all sequences
    int c = max(first - tile, 0);
    for (int b = 32 + lane; b < a.batch; b += 32) c += max(tiles_of(b) - tile, 0);
    return __reduce_add_sync(0xFFFFFFFFu, c);
  };
  int at = x / a.hkv, tile = 0, after = 0;  // after: tiles behind `tile`
  u.head = x % a.hkv;
  if (at >= count(0)) return false;
  for (int end = a.tiles; end - tile > 1;) {
    const int mid = (tile + end) / 2, c = count(mid);
    if (c > at) tile = mid;
    else end = mid, after = c;
  }
  at -= after;
  u.b = -1;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const bool has = (b0 ? tiles_of(b0 + lane) : first) > tile;
    const uint32_t m = __ballot_sync(0xFFFFFFFFu, has);
    const uint32_t me = __ballot_sync(0xFFFFFFFFu, has && __popc(m & ((1u << lane) - 1)) == at);
    if (me) {
      u.b = b0 + __ffs(me) - 1;
      break;
    }
    at -= __popc(m);
  }
  if (u.b < 0) return false;
  const bool early = u.b < 32;
  u.q0 = early ? __shfl_sync(0xFFFFFFFFu, start, u.b & 31) : a.starts[u.b];
  const int n = early ? __shfl_sync(0xFFFFFFFFu, given, u.b & 31) : a.starts[u.b + 1] - u.q0;
  const int64_t len = early ? __shfl_sync(0xFFFFFFFFu, held, u.b & 31) : a.lens[u.b];
  u.n = new_tokens(a, u.q0, n);
  u.t0 = tile * per;
  if (u.t0 >= u.n) return false;  // the lengths changed under the kernel
  u.len = static_cast<int>(len < 0 ? 0 : len > a.room ? a.room : len);
  u.base = u.len - n;
  const int end = u.base + min(u.n, u.t0 + per);  // one past the last query's position
  u.lo = a.window > 0 ? max(0, u.base + u.t0 - a.window + 1) : 0;
  u.all = end > 0 ? (end + C::BN - 1) / C::BN - u.lo / C::BN : 0;
  u.share = a.splits > 1 ? max((u.all + a.splits - 1) / a.splits, kMinShare) : max(u.all, 1);
  return true;
}

// What the warp that loads tells the others of the CTA's next work.
struct alignas(16) Plan {
  int more;                        // 0: there is none
  int rows, b, head, q0, n, base;  // rows: first of the partials; the rest as in Unit
  int len, t0, lo, j0, nt, parts;  // key tiles j0 to j0 + nt; parts: others have more of them
  int pad[3];
};
static_assert(sizeof(Plan) == 64, "of shared memory");

// A [tokens][64 columns] block of 128-byte rows read with the columns as the long (N)
// dimension: 64-column blocks `block` bytes apart, groups of 8 tokens `group` apart.
__device__ __forceinline__ uint64_t umma_smem_desc_mn(uint32_t saddr, uint32_t block, uint32_t group) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(block >> 4) << 16;
  d |= static_cast<uint64_t>(group >> 4) << 32;
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
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
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

// ---- pairs of 32-bit values in one instruction --------------------------------------------
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The larger of two, of three, NaN if one is.
__device__ __forceinline__ float fmaxf_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The weights 2^(s * s2 - z) of N scores, packed to 16 bits, their sum added to `sum`.
template <int DT, int N>
__device__ __forceinline__ void weights(const float* s, float s2, float z, uint32_t* p, uint64_t* sum) {
  const uint64_t k = pair(s2, s2), nz = pair(-z, -z);
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    float a, b;
    unpair(fma2(pair(s[2 * c], s[2 * c + 1]), k, nz), a, b);
    a = exp2_fast(a);
    b = exp2_fast(b);
    sum[c & 1] = add2(sum[c & 1], pair(a, b));
    // rounded to the cache's type for the product, whose two operands have one type; the sum is
    // not. That adds as much as the output's own rounding: relative error against 64 bits 0.0019 to
    // 0.0022 in bf16 where 32-bit weights give 0.0016
    p[c] = pack16<DT>(a, b);
  }
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

struct alignas(16) Answer {
  long long x, y;
};

template <int DP, int QT, int DT>
__global__ void __launch_bounds__(PShape<DP, QT>::THREADS, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap vmap,
                        const __grid_constant__ PromptArgs a) {
  using C = PShape<DP, QT>;
  constexpr int NQ = C::NQ, BN = C::BN, NB = C::NB, SLOTS = C::SLOTS, OW = C::OW;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sq = smem;
  uint8_t* ring = sq + NQ * C::QB;  // K(0), V(0), K(1), V(1), ... in turn
  uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + C::BARS);
  uint64_t* qfree = qfull + 1;    // the queries have been multiplied
  uint64_t* full = qfree + 1;
  uint64_t* empty = full + SLOTS;
  uint64_t* vfix = empty + SLOTS;
  uint64_t* sfree = vfix + 1;     // the score buffer's content is in registers
  uint64_t* told = sfree + 1;     // the plan is there
  uint64_t* heard = told + 1;     // it has been read
  uint64_t* next = heard + 1;     // the answer to the question for another unit
  uint64_t* drained = next + 1;   // after a wait that ran out: the products issued until then are done
  uint64_t* sfull = drained + 1;  // [NQ] a query tile's scores are in the buffer
  uint64_t* odone = sfull + NQ;   // [NQ] a query tile's product with the values is done
  uint64_t* ofree = odone + NQ;   // [NQ] a query tile's output has been read
  uint64_t* pready = ofree + NQ;  // [NQ][2] half of a query tile's weights
  static_assert(8 + 2 * SLOTS + 5 * NQ == C::NBARS, "the barriers above");
  Plan* plan = reinterpret_cast<Plan*>(smem + C::PLAN);
  uint4* answer = reinterpret_cast<uint4*>(plan + 1);
  uint32_t* slot = reinterpret_cast<uint32_t*>(answer + 1);
  // the same in all lanes, and known to be: the products' operands then live in uniform registers
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {  // the swizzled tiles need it, and a CTA's memory starts so
    if (threadIdx.x == 0) atomicOr(&g_device_error, kErrIndex);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(qfull, 1);
    mbar_init(qfree, 1);
    for (int i = 0; i < SLOTS; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
    mbar_init(vfix, 1);
    mbar_init(sfree, 4);
    mbar_init(told, 1);
    mbar_init(heard, 3 + 4 * NQ);
    mbar_init(next, 1);
    mbar_init(drained, 1);
    for (int i = 0; i < NQ; ++i) mbar_init(sfull + i, 1), mbar_init(odone + i, 1), mbar_init(ofree + i, 4);
    for (int i = 0; i < 2 * NQ; ++i) mbar_init(pready + i, 4);
    fence_mbar_init();
  }
  pdl_wait();
  Unit u;
  bool some = false;
  if (warp == OW) some = unit_of<DP, QT>(a, static_cast<int>(blockIdx.x), u);
  if (warp == OW + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(static_cast<uint32_t>(C::COLS))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *slot, 0);
  // not earlier: a dependent kernel that takes its tensor memory before it waits for this
  // grid must find that all of this grid's CTAs have theirs
  pdl_trigger();

  auto warp_wait = [](uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity)) != 0; };
  // every other warp: the next plan; false where a wait ran out
  auto hear = [&](Plan& p, int count) {
    const bool ok = mbar_wait(told, count & 1);
    if (!__all_sync(0xFFFFFFFFu, ok)) return false;
    p = *plan;
    __syncwarp();
    if (lane == 0) mbar_arrive(heard);
    return true;
  };

  // the softmax warps hold a row's scores in registers: they take what the others leave
  // (208 + 208 + 88 = 3 x 168, the launch's share)
  if (warp >= OW) {
    if (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == OW) {
      // ---- what to do next; queries and values, by TMA ---------------------------------------
      // a lane's box of a tile: all column blocks of box rows, or one of them; and its page
      const int cols = a.one_box ? 1 : NB, boxes = cols * (BN / a.box), rb = lane / cols, cb = lane % cols;
      bool ok = true;
      int x = static_cast<int>(blockIdx.x), split = static_cast<int>(blockIdx.y);
      int plans = 0, works = 0, tiles = 0, fixes = 0, sl = 1;  // plans told, with key tiles; tiles loaded in all
      uint32_t par = 1, asked = 0;
      auto tell = [&](const Plan& p) {
        if (plans) ok = mbar_wait(heard, (plans - 1) & 1);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) return;
        if (lane == 0) {
          *plan = p;
          mbar_arrive(told);
        }
        __syncwarp();
        ++plans;
      };
      for (;;) {
        Plan p;
        if (some) {
          p = {1,     a.splits > 1 ? (x * a.splits + split) * (NQ * 128) : 0, u.b, u.head, u.q0, u.n, u.base, u.len, u.t0, u.lo,
               u.lo / BN + split * u.share, min(u.share, u.all - split * u.share), u.all > u.share, {}};
          some = p.parts || split == 0;
        }
        if (some) tell(p);
        if (some && ok && p.nt > 0) {
          if (works) ok = mbar_wait(qfree, (works - 1) & 1);
          if (!__all_sync(0xFFFFFFFFu, ok)) break;
          if (lane == 0) mbar_arrive_expect_tx(qfull, NQ * NB * a.toks * a.group * 128);
          __syncwarp();
          if (lane < NQ * NB) {
            const int i = lane / NB, c = lane % NB;
            tma_load_4d(sq + i * C::QB + c * (128 * 128), &qmap, c * 64, 0, p.head, p.q0 + p.t0 + i * a.toks, qfull);
          }
          ++works;
          const int32_t* row = a.tables + p.b * a.table_row;
          auto page_of = [&](int j) {
            const int tok = j * BN + rb * a.box;
            if (lane >= boxes || tok >= p.len || tok + a.box <= p.lo) return a.num_pages;  // the box is filled with zeros
            const int pg = row[tok / a.page_size];
            if (pg >= 0 && pg < a.num_pages) return pg;
            atomicOr(&g_device_error, kErrIndex);
            return a.num_pages;
          };
          auto load = [&](uint8_t* dst, int j, int page, uint64_t* bar) {
            if (lane == 0) mbar_arrive_expect_tx(bar, C::KB);
            __syncwarp();
            if (lane < boxes)
              tma_load_5d(dst + (a.one_box ? rb * (a.box * NB * 128) : cb * (BN * 128) + rb * (a.box * 128)), &vmap, cb * 64,
                          (j * BN + rb * a.box) % a.page_size, 0, p.head, page, bar);
          };
          int page = page_of(p.j0);  // the values have every other tile of the ring
          for (int t = 0; t < p.nt; ++t) {
            const int j = p.j0 + t, later = t + 1 < p.nt ? page_of(j + 1) : 0;
            ok = mbar_wait(empty + sl, par);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            uint8_t* dst = ring + sl * C::KB;
            // tokens past the length that share a box with some before it may hold anything, NaN
            // too, and a weight of 0 must meet 0: that tile's values are cleared there by hand
            if ((j + 1) * BN > p.len && p.len % a.box) {
              load(dst, j, page, vfix);
              ok = mbar_wait(vfix, fixes++ & 1);
              ok = __all_sync(0xFFFFFFFFu, ok);
              if (!ok) break;
              const int r0 = p.len - j * BN, rows = (r0 + a.box - 1) / a.box * a.box - r0;
              for (int x8 = lane; x8 < rows * NB * 8; x8 += 32) {
                const int c = x8 / 8 % NB, r = r0 + x8 / 8 / NB;
                const int at = a.one_box ? (r / a.box * NB + c) * (a.box * 128) + r % a.box * 128 : c * (BN * 128) + r * 128;
                *reinterpret_cast<uint4*>(dst + at + x8 % 8 * 16) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(full + sl);
            } else {
              load(dst, j, page, full + sl);
            }
            page = later;
            ++tiles;
            sl += 2;
            if (sl >= SLOTS) sl -= SLOTS, par ^= 1;
          }
        }
        if (!ok) break;
        // another unit, one that no CTA has begun; not earlier, since a free CTA would begin it sooner
        if (lane == 0) {
          mbar_arrive_expect_tx(next, 16);
          cuda::ptx::clusterlaunchcontrol_try_cancel(answer, next);
        }
        __syncwarp();
        // (mbar_wait's own polls may each pause for longer than any wait in here takes: a limit on those
        // does not make one run out)
        ok = a.polls ? mbar_poll(next, asked & 1, a.polls) : mbar_wait(next, asked & 1);
        ++asked;
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        const longlong2 got = *reinterpret_cast<const longlong2*>(answer);
        const Answer ans{got.x, got.y};
        if (!cuda::ptx::clusterlaunchcontrol_query_cancel_is_canceled(ans)) {
          p = {};
          tell(p);
          break;
        }
        x = cuda::ptx::clusterlaunchcontrol_query_cancel_get_first_ctaid_x<int>(ans);
        split = cuda::ptx::clusterlaunchcontrol_query_cancel_get_first_ctaid_y<int>(ans);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read before it is written again
        __syncwarp();
        some = unit_of<DP, QT>(a, x, u);
      }
      if (blockIdx.x == 0 && blockIdx.y == 0)  // lengths that do not fit
        for (int b = lane; b < a.batch; b += 32) {
          const int q0 = a.starts[b], n = a.starts[b + 1] - q0;
          if (n < 0 || n > new_tokens(a, q0, n) || a.lens[b] > a.room) atomicOr(&g_device_error, kErrIndex);
        }
      if (!ok) {  // a wait ran out: the copies and the answer still in flight
        if (works) mbar_drain(qfull, (works - 1) & 1);
        for (int t = max(0, tiles - 1 - SLOTS / 2); t < tiles; ++t)
          mbar_drain(full + (2 * t + 1) % SLOTS, (2 * t + 1) / SLOTS & 1);
        if (fixes) mbar_drain(vfix, (fixes - 1) & 1);
        if (asked) mbar_drain(next, (asked - 1) & 1);
      }
    } else if (warp >= OW + 2) {
      // ---- keys, two warps in turn, by 16-byte copies: a TMA box of one 64-column block of a
      // 16-token page is a request of 2 KB, and the unit takes about 134 clocks for each
      constexpr int CH = DP / 8, RPI = 32 / CH;  // 16-byte chunks of a row, rows of a warp's copy
      const int ch = lane % CH, sub = lane / CH;
      const bool col = ch * 8 < a.d;
      const uint32_t dst0 = smem_u32(ring) + (ch >> 3) * (BN * 128);
      Plan p;
      bool ok = true;
      for (int plans = 0, tiles = 0; ok && hear(p, plans) && p.more; ++plans) {
        if (p.nt <= 0) continue;
        const int32_t* row = a.tables + p.b * a.table_row;
        const uint16_t* base = a.k + p.head * a.k_head + (col ? ch * 8 : 0);
        // lane x: where tokens 8 x .. 8 x + 7 of a tile lie, negative where they are not read
        auto place_of = [&](int j) -> int64_t {
          const int tok = j * BN + lane * 8;
          if (lane >= BN / 8 || tok >= p.len || tok + 8 <= p.lo) return -1;
          const int pg = row[tok / a.page_size];
          if (pg < 0 || pg >= a.num_pages) return -1;  // reads as zeros; the values' warp reports it
          return pg * a.k_page + tok % a.page_size * a.k_slot;
        };
        int t = (warp - OW - 2) ^ (tiles & 1);
        int64_t place = place_of(p.j0 + t);
        for (; t < p.nt; t += 2) {
          const int64_t later = t + 2 < p.nt ? place_of(p.j0 + t + 2) : 0;
          const int at2 = 2 * (tiles + t), sl = at2 % SLOTS;  // the keys have every other tile of the ring
          ok = mbar_wait(empty + sl, (at2 / SLOTS & 1) ^ 1);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          const uint32_t dst = dst0 + sl * C::KB;
#pragma unroll 4
          for (int g = 0; g < BN / 8; ++g) {
            const int64_t at = __shfl_sync(0xFFFFFFFFu, place, g);
            const bool in = at >= 0 && col;
            const uint16_t* src = in ? base + at : a.k;
            const int64_t step = in ? a.k_slot : 0;
            const uint32_t bytes = in ? 16 : 0;  // the rest of the 16 is filled with zeros
#pragma unroll
            for (int x = 0; x < 8; x += RPI) {
              const int r = x + sub;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (g * 8 + r) * 128 +
                                                                                (((ch & 7) ^ r) << 4)),
                           "l"(src + r * step), "r"(bytes)
                           : "memory");
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(full + sl);
          place = later;
        }
        tiles += p.nt;
      }
    } else if (warp == OW + 1) {
      // ---- products --------------------------------------------------------------------
      // the whole warp walks the tiles, one elected lane issues; all lanes agree on how a wait ended,
      // or some would miss where the others elect
      constexpr uint32_t id_qk = idesc16<DT, BN, false>(), id_pv = idesc16<DT, DP, true>();
      // a V tile: boxes of all column blocks one after the other, or one block after the other
      const uint32_t vblock = a.one_box ? a.box * 128 : BN * 128;
      const uint32_t vgroup = a.one_box && a.box == 8 ? NB * 1024 : 1024;
      const uint32_t vlog = __ffs(a.box) - 1;
      const uint32_t vbox = a.one_box ? a.box * NB * 128 : a.box * 128;  // from box to box
      const uint64_t q_desc = umma_smem_desc(smem_u32(sq)), k_desc = umma_smem_desc(smem_u32(ring));
      const uint64_t v_desc = umma_smem_desc_mn(smem_u32(ring), vblock, vgroup);
      uint32_t v_at[BN / 16];  // of each 16 tokens of a tile, in units of 16 bytes
#pragma unroll
      for (int k = 0; k < BN / 16; ++k)
        v_at[k] = ((16u * k >> vlog) * vbox + (16u * k & ((1u << vlog) - 1)) * 128) >> 4;
      int tiles = 0, works = 0;              // key tiles of the units before, and those units
      auto qk = [&](int i, int t, int sl) {  // scores of query tile i, key tile t
        const int use = (tiles + t) * NQ + i;  // of the score buffer: the one before must be in registers
        if (use && !warp_wait(sfree, (use - 1) & 1)) return false;
        fence_after();
        const uint64_t qd = q_desc + i * (C::QB >> 4), kd = k_desc + static_cast<uint32_t>(sl * (C::KB >> 4));
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < NB; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ss(tmem, qd + (c * (128 * 128 >> 4) + 2 * k), kd + (c * (BN * 128 >> 4) + 2 * k), id_qk, c > 0 || k > 0);
          umma_commit(sfull + i);
        }
        __syncwarp();
        return true;
      };
      // the output of query tile i takes a value tile; the first half of the weights may be
      // multiplied while the second is still being made
      auto pv = [&](int i, int t, int sl) {
        const uint64_t vd = v_desc + static_cast<uint32_t>(sl * (C::KB >> 4));
        if (t == 0 && works && !warp_wait(ofree + i, (works - 1) & 1)) return false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!warp_wait(pready + i * 2 + h, (tiles + t) & 1)) return false;
          fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = h * (BN / 32); k < (h + 1) * (BN / 32); ++k)
              umma_ts(tmem + C::OCOL + i * DP, tmem + C::PCOL + i * (BN / 2) + 8 * k, vd + v_at[k], id_pv, t > 0 || k > 0);
            if (h) umma_commit(odone + i);
          }
          __syncwarp();
        }
        return true;
      };
      int sl = 0;  // the ring's next slot and its parity
      uint32_t par = 0;
      auto wait_tile = [&](int& at) {  // the next tile of the ring has arrived
        at = sl;
        const bool ok = warp_wait(full + sl, par);
        fence_after();
        if (++sl == SLOTS) sl = 0, par ^= 1;
        return ok;
      };
      auto release = [&](int at) {
        if (elect_one()) umma_commit(empty + at);
        __syncwarp();
      };
      Plan p;
      bool ok = true;
      for (int plans = 0; ok; ++plans) {
        ok = hear(p, plans);
        if (!ok || !p.more) break;
        const int nt = p.nt;
        if (nt <= 0) continue;
        int ks = 0, vs = 0;
        auto queries_done = [&]() {
          if (elect_one()) umma_commit(qfree);
          __syncwarp();
        };
        ok = warp_wait(qfull, works & 1) && wait_tile(ks);
        for (int i = 0; i < NQ; ++i) ok = ok && qk(i, 0, ks);
        if (ok) release(ks);
        if (ok && nt == 1) queries_done();
        for (int t = 0; t < nt && ok; ++t) {
          const bool more = t + 1 < nt;
          ok = wait_tile(vs);
          if (ok && more) ok = wait_tile(ks);
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if (more) {
              ok = ok && qk(i, t + 1, ks);
              if (ok && i == NQ - 1) {
                release(ks);
                if (t + 2 == nt) queries_done();
              }
            }
            ok = ok && pv(i, t, vs);
          }
          if (ok) release(vs);
        }
        tiles += nt;
        ++works;
      }
      if (!ok) {  // a wait ran out: the products still in flight read and write this CTA's memory
        if (elect_one()) umma_commit(drained);
        __syncwarp();
        mbar_drain(drained, 0);
      }
    }
  } else {
    if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: thread r of a warpgroup has row r of its query tile ---------------------
    const int i = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    // 16-bit floats underflow early (2^-24), and a long tail of small weights can add up: theirs
    // are kept 2^11 larger, the sum too, and rescaled when the maximum has grown by 2^4
    constexpr float kUp = DT == GGUFMM_F16 ? 11.f : 0.f, kGrow = DT == GGUFMM_F16 ? 4.f : 8.f;
    const bool odd_scale = a.s2 <= 0.f;
    const float s2 = odd_scale ? 1.f : a.s2;
    float* const part_ml = a.part + static_cast<int64_t>(a.units) * a.splits * (NQ * 128) * DP;
    const int mine = i * a.toks + r / a.group, g = r % a.group;  // token and head
    // whole sectors, where the rows begin on them: half the requests, which bound the output's writing
    const bool wide = (a.o_row | a.o_head | a.d) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 32 == 0;
    bool ok = true;
    Plan p;
    for (int plans = 0, tiles = 0; ok && hear(p, plans) && p.more; ++plans) {
      uint16_t* const outp = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(p.head) * a.group * a.o_head;
      const int nt = p.nt;
      if (nt <= 0 && p.parts) {  // nothing of the unit is left for this CTA
        *reinterpret_cast<float2*>(part_ml + (static_cast<int64_t>(p.rows) + i * 128 + r) * 2) = make_float2(-INFINITY, 0.f);
        continue;
      }
      if (nt <= 0) {  // every query lies before position 0
        const int c8 = a.d / 8, cnt = min(NQ * a.toks, p.n - p.t0) * a.group * c8;
        for (int e = threadIdx.x; e < cnt; e += NQ * 128) {
          const int c = e % c8, h = e / c8 % a.group, t = e / c8 / a.group;
          *reinterpret_cast<uint4*>(outp + static_cast<int64_t>(p.q0 + p.t0 + t) * a.o_row + h * a.o_head + c * 8) =
              make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      const int tok = p.t0 + mine;
      const bool live = r < a.toks * a.group && tok < p.n;
      const int pos = p.base + tok;  // this row's position
      const int pos_a = p.base + p.t0 + i * a.toks, pos_b = pos_a + a.toks - 1;  // the tile's first and last
      const int j0 = p.j0;
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < nt; ++t) {
        ok = mbar_wait(sfull + i, (tiles + t) & 1);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        fence_after();
        uint32_t sr[BN];
#pragma unroll
        for (int c = 0; c < BN; c += 32) tmem_ld32(lanes + c, sr + c);
        tmem_wait_ld();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sfree);
        float* s = reinterpret_cast<float*>(sr);
        if (odd_scale) {
#pragma unroll
          for (int c = 0; c < BN; ++c) s[c] *= a.s2;
        }
        const int jb = (j0 + t) * BN;
        const bool edge = jb + BN - 1 > pos_a || (a.window > 0 && jb <= pos_b - a.window);
        if (edge) {
          const int up = pos - jb, dn = a.window > 0 ? pos - a.window - jb : -1;  // visible: dn < c <= up
#pragma unroll
          for (int c = 0; c < BN; ++c)
            if (c > up || c <= dn) s[c] = -INFINITY;
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(s[e], s[4 + e], s[8 + e]);
#pragma unroll
        for (int c = 12; c + 8 <= BN; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
        static_assert((BN - 12) % 8 == 4, "the last four");
        mx[0] = max3(mx[0], s[BN - 4], s[BN - 3]);
        mx[1] = max3(mx[1], s[BN - 2], s[BN - 1]);
        // a row of no token of this sequence holds anything, and has no say in rescaling
        const float top = live ? max3(fmaxf_nan(mx[0], mx[1]), mx[2], mx[3]) * s2 : -INFINITY;
        // rescale when the maximum has grown by more than kGrow (or is the first; a NaN stays one)
        float f = 1.f;
        if (!(top <= m + kGrow)) {
          f = exp2_fast(m - top);  // 0 for the first
          m = top == INFINITY ? __int_as_float(0x7FFFFFFF) : top;  // inf - inf
          l *= f;
        }
        if (t > 0) {  // the product that reads the last weights, and adds to the output
          ok = mbar_wait(odone + i, (tiles + t - 1) & 1);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          fence_after();
        }
        if (t > 0 && __any_sync(0xFFFFFFFFu, f != 1.f)) {
          const uint32_t oc = lanes + C::OCOL + i * DP;
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tmem_ld32(oc + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(oc + c, o);
            tmem_st16(oc + c + 16, o + 16);
          }
        }
        const float z = (m == -INFINITY ? 0.f : m) - kUp;
        uint64_t sum[2] = {0, 0};
        auto handed = [&](int h) {  // half h of the weights is in tensor memory
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pready + i * 2 + h);
        };
        const uint32_t pc = lanes + C::PCOL + i * (BN / 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[BN / 4];
          const float* v = s + h * (BN / 2);
          weights<DT, BN / 2>(v, s2, z, w, sum);
          if (h) handed(0);  // its store has had time to finish
#pragma unroll
          for (int c = 0; c < BN / 4; c += 16) tmem_st16(pc + h * (BN / 4) + c, w + c);
        }
        handed(1);
        float a0, a1;
        unpair(add2(sum[0], sum[1]), a0, a1);
        l += a0 + a1;
      }
      tiles += nt;
      if (ok) ok = mbar_wait(odone + i, (tiles - 1) & 1);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (ok) {
        fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* dst = outp + static_cast<int64_t>(p.q0 + tok) * a.o_row + g * a.o_head;
        const uint32_t oc = lanes + C::OCOL + i * DP;
        const int64_t pr = static_cast<int64_t>(p.rows) + i * 128 + r;
        float* po = a.part + pr * DP;
        if (p.parts) *reinterpret_cast<float2*>(part_ml + pr * 2) = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(oc + c, o);
          tmem_wait_ld();
          if (p.parts) {
            if (live) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) store32(po + c + e, o + e);
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              if (c + e >= a.d) break;
              uint32_t w[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float v0 = l == 0.f ? 0.f : __uint_as_float(o[e + 2 * x]) * inv;
                const float v1 = l == 0.f ? 0.f : __uint_as_float(o[e + 2 * x + 1]) * inv;
                w[x] = pack16<DT>(v0, v1);
              }
              if (wide) {
                store32(dst + c + e, w);
              } else {
                *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
                if (c + e + 8 < a.d) *reinterpret_cast<uint4*>(dst + c + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
              }
            }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ofree + i);
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == OW + 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(static_cast<uint32_t>(C::COLS))
                 : "memory");
  }
}

// Adds the splits' partials of a row, in their order: one warp a row.
template <int DP, int QT, int DT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ PromptArgs a) {
  using C = PShape<DP, QT>;
  constexpr int R = C::NQ * 128, V = DP / 32;  // rows of a unit, values of a lane
  __shared__ Unit un;
  __shared__ int parts;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, r = static_cast<int>(blockIdx.y) * 8 + (threadIdx.x >> 5);
  if (threadIdx.x < 32) {
    Unit u;
    const bool some = unit_of<DP, QT>(a, static_cast<int>(blockIdx.x), u);
    if (lane == 0) {
      if (some) un = u;
      parts = some && u.all > u.share;
    }
  }
  __syncthreads();
  if (!parts) return;  // nothing, or written by one CTA
  const int in = r % 128, tok = un.t0 + r / 128 * a.toks + in / a.group, g = in % a.group;
  if (in >= a.toks * a.group || tok >= un.n) return;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.splits * R + r;
  const float* ml = a.part + static_cast<int64_t>(a.units) * a.splits * R * DP;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[(row0 + static_cast<int64_t>(s) * R) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const float z = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[V] = {};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const int64_t row = row0 + static_cast<int64_t>(s) * R;
    const float2 w = *reinterpret_cast<const float2*>(ml + row * 2);
    if (w.x == -INFINITY) continue;  // it saw nothing, and wrote no output
    const float f = exp2_fast(w.x - z);
    l += w.y * f;
#pragma unroll
    for (int c = 0; c < V; c += 2) {
      const float2 v = *reinterpret_cast<const float2*>(a.part + row * DP + (c / 2) * 64 + lane * 2);
      acc[c] += v.x * f;
      acc[c + 1] += v.y * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(un.q0 + tok) * a.o_row +
                  (static_cast<int64_t>(un.head) * a.group + g) * a.o_head;
#pragma unroll
  for (int c = 0; c < V; c += 2) {
    const int col = (c / 2) * 64 + lane * 2;
    if (col < a.d)
      *reinterpret_cast<uint32_t*>(dst + col) =
          pack16<DT>(l == 0.f ? 0.f : acc[c] * inv, l == 0.f ? 0.f : acc[c + 1] * inv);
  }
}

std::atomic<uint32_t> lowered_polls{0};  // ggufmm_set_wait_limit's, 0 where it is not lowered

// How the work of a call is cut: query tiles per sequence, CTAs for them, and, where those
// leave SMs idle and the cache may be long, shares of the keys for several CTAs each.
struct Cut {
  int nq, tiles, units, splits, rows, dp;
  size_t bytes() const { return splits > 1 ? static_cast<size_t>(units) * splits * rows * (dp + 2) * 4 : 0; }
};
Cut cut_of(const ggufmm_attention_args& p, int sms) {
  Cut c;
  c.dp = p.head_dim <= 64 ? 64 : p.head_dim <= 128 ? 128 : 256;
  const int64_t one = 128 / (p.q_heads / p.kv_heads);
  c.nq = c.dp == 256 || p.max_q <= one ? 1 : 2;
  const int nq = c.nq, bn = c.dp == 256 ? PShape<256, 1>::BN : PShape<128, 2>::BN;
  const int64_t toks = nq * one;
  const int64_t tiles = (p.max_q + toks - 1) / toks;
  const int64_t units = std::min(tiles * p.batch, (p.total_q + p.batch * (toks - 1)) / toks) * p.kv_heads;  // at most
  c.tiles = static_cast<int>(tiles);
  c.units = static_cast<int>(units);
  c.rows = nq * 128;
  int64_t longest = (p.table_width * p.page_size + bn - 1) / bn;
  if (p.window > 0) longest = std::min<int64_t>(longest, (p.window + toks + bn - 1) / bn + 1);
  c.splits = units >= sms ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / units, longest / kMinShare)));
  return c;
}

bool encode(CUtensorMap* map, int64_t dtype, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  PFN_encodeTiled enc = get_encode_fn();
  if (!enc) return false;
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(map, dtype == GGUFMM_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
             static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int QT, int DT>
cudaError_t launch(const ggufmm_attention_args& p, const Cut& cut, void* workspace, cudaStream_t st) {
  using C = PShape<DP, QT>;
  const cuuint64_t d = static_cast<cuuint64_t>(p.head_dim), g = static_cast<cuuint64_t>(p.q_heads / p.kv_heads);
  PromptArgs a;
  a.out = p.out;
  a.tables = static_cast<const int32_t*>(p.tables);
  a.lens = static_cast<const int32_t*>(p.lens);
  a.starts = static_cast<const int32_t*>(p.q_starts);
  a.k = static_cast<const uint16_t*>(p.k);
  a.k_page = p.k_page;
  a.k_head = p.k_head;
  a.k_slot = p.k_slot;
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
  a.tiles = cut.tiles;
  a.units = cut.units;
  a.splits = cut.splits;
  a.part = static_cast<float*>(workspace);
  a.d = static_cast<int>(p.head_dim);
  a.page_size = static_cast<int>(p.page_size);
  a.num_pages = static_cast<int>(p.num_pages);
  a.window = p.window < a.room ? static_cast<int>(p.window) : 0;  // one as wide as the table hides nothing
  a.s2 = static_cast<float>(p.scale * 1.4426950408889634);
  a.polls = lowered_polls.load(std::memory_order_relaxed);
  a.box = 8;  // the largest run of rows up to a tile that divides a page
  while (a.box < C::BN && p.page_size % (2 * a.box) == 0) a.box *= 2;
  CUtensorMap qm, vm;
  const cuuint64_t qd[4] = {d, g, static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.total_q)};
  const cuuint64_t qs[3] = {static_cast<cuuint64_t>(p.q_head) * 2, static_cast<cuuint64_t>(p.q_head) * g * 2,
                            static_cast<cuuint64_t>(p.q_row) * 2};
  const cuuint32_t qb[4] = {64, static_cast<cuuint32_t>(g), 1, static_cast<cuuint32_t>(a.toks)};
  // the values with their 64-column blocks as a dimension of its own, so that one box of
  // whole rows takes half (a quarter of) the requests: with pages of 16 tokens the loads
  // are bound by those
  a.one_box = a.d == DP;
  const cuuint64_t blocks = a.one_box ? C::NB : 1;
  const cuuint64_t vd[5] = {a.one_box ? 64 : d, static_cast<cuuint64_t>(p.page_size), blocks,
                            static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.num_pages)};
  const cuuint64_t vs[4] = {static_cast<cuuint64_t>(p.v_slot) * 2, 128, static_cast<cuuint64_t>(p.v_head) * 2,
                            static_cast<cuuint64_t>(p.v_page) * 2};
  const cuuint32_t vb[5] = {64, static_cast<cuuint32_t>(a.box), static_cast<cuuint32_t>(blocks), 1, 1};
  if (!encode(&qm, p.dtype, p.q, 4, qd, qs, qb) || !encode(&vm, p.dtype, p.v, 5, vd, vs, vb)) return cudaErrorInvalidValue;
  auto fn = paged_prompt_kernel<DP, QT, DT>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  if (!(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return e;
    // the warps' shares of registers must add up to no more than the launch brings: a build
    // that needs fewer would wait for registers that nobody gives back
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, fn);
    if (e != cudaSuccess) return e;
    if (C::NQ == 2 && fa.numRegs < kLaunchRegs) return cudaErrorInvalidKernelImage;
    ready.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_release);
  }
  e = pdl_launch(fn, dim3(static_cast<unsigned>(a.units), static_cast<unsigned>(a.splits)), dim3(C::THREADS), C::SMEM, st, qm,
                 vm, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  return pdl_launch(join_kernel<DP, QT, DT>, dim3(static_cast<unsigned>(a.units), C::NQ * 16), dim3(256), 0, st, a);
}

}  // namespace

size_t paged_prompt_workspace(const ggufmm_attention_args& p, int sms) { return cut_of(p, sms).bytes(); }

cudaError_t launch_paged_prompt(const ggufmm_attention_args& p, int sms, void* workspace, size_t workspace_bytes,
                                cudaStream_t st) {
  Cut cut = cut_of(p, sms);
  if (!workspace || workspace_bytes < cut.bytes()) cut.splits = 1;
  const bool f16 = p.dtype == GGUFMM_F16;
  auto sized = [&](auto dp, auto qt) {
    constexpr int DP = decltype(dp)::value, QT = decltype(qt)::value;
    return f16 ? launch<DP, QT, GGUFMM_F16>(p, cut, workspace, st) : launch<DP, QT, GGUFMM_BF16>(p, cut, workspace, st);
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  if (cut.dp == 64) return cut.nq == 1 ? sized(std::integral_constant<int, 64>{}, one) : sized(std::integral_constant<int, 64>{}, two);
  if (cut.dp == 128)
    return cut.nq == 1 ? sized(std::integral_constant<int, 128>{}, one) : sized(std::integral_constant<int, 128>{}, two);
  return sized(std::integral_constant<int, 256>{}, one);
}

cudaError_t attn_prompt_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }
cudaError_t attn_prompt_set_wait_limit(uint32_t polls) {
  lowered_polls.store(polls < kWaitLimit ? polls : 0, std::memory_order_relaxed);
  return tu_set_wait_limit(polls);
}

}  // namespace ggufmm
