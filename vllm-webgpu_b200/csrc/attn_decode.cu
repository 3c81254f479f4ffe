// attn_decode.cu -- ggufmm_paged_attention: attention of one new token per sequence over
// the paged key-value cache, the cache's length split over the SMs and joined in the same
// launch.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q.k_j,  m = max_j s_j
//
// One pass over the keys and values with a running m and sum. The G = q_heads / kv_heads
// query heads that share a kv head are the rows of one 16-row tensor-core tile, so each
// cached value is read once (once per 16 of them where G is larger: the parts are items of their
// own): 2 G flops per byte, far below what the tensor cores need, and the time is the cache's
// bytes over the HBM rate.
//
// Split: the work is the list of all (sequence, kv head) items, cut into blocks of W * 16
// tokens; an item counts as one block more, for what it costs to begin and to end one. Every
// CTA (one per SM) takes an equal run of consecutive blocks, whatever sequences they belong
// to, so ragged lengths leave no SM idle; it finds its run by a sum over the lengths on the
// device. An item inside one run is written directly. An item that crosses runs leaves fp32
// partials (m, sum, o) in the workspace, and the last of its CTAs to finish (a counter) adds
// them in the order of the CTAs, so the result does not depend on which was last. (Handing part of the work out in short runs as CTAs finish was measured:
// 196 to 208 us for 64 sequences up to 8192 tokens against 195, 124 to 152 us for one of 131035
// against 105, since every run costs a join.)
//
// Inside a CTA each warp owns every W-th group of 16 tokens and its own ring of stages, filled
// by 16-byte asynchronous copies S groups ahead of use, across items: no barrier between warps
// except where an item ends, and the ring keeps streaming over that too. (TMA boxes of whole
// 16-token pages did as well at head width 128, but the unit takes about 134 clocks for every
// request: pages of 8 or 24 tokens, or heads that are no multiple of 64 wide, got 2.4 TB/s.)
//
// 32 / 8 heads of 128, bf16, pages of 16: 64 sequences up to 8192 tokens (1.155 GB) 184 us, 6.27
// TB/s, 97% of the measured copy rate; 16 around 1300 (90 MB) 25 us; one of 513 9.1 us. 64 / 8 heads,
// f16, one sequence of 131035 (537 MB) 94 us, 5.7 TB/s; 64 of up to 8192 with a window of 1024
// (270 MB) 52 us, 5.2 TB/s; 32 of up to 4096, 32 heads to one kv head (63 MB read twice) 31.5 us;
// 8 / 2 heads of 256 (251 MB) 56 us, 4.5 TB/s. HBM bound when long; when short the time is
// a chain of waits: lengths, page table, first copies (4 us), join in the CTA (0.8), join of CTAs (1.5).
#include <algorithm>
#include <atomic>
#include <cmath>

#include "mma16.cuh"
#include "paged.cuh"

namespace ggufmm {

struct DevInfo {
  int sms = 0;
  int smem_optin = 0;
};
DevInfo device_info(int dev);  // capi.cu

namespace {

constexpr int kMaxGrid = 160;               // CTAs a workspace has room for
constexpr size_t kCounterBytes = 1024;      // one arrival counter per CTA
static_assert(kMaxGrid * 4 <= kCounterBytes, "counters");

template <int DP>
struct Shape {
  static constexpr int W = DP == 256 ? 4 : 8;       // warps
  static constexpr int HALF = 16 * DP * 2;          // bytes of 16 tokens of K (or V)
  static constexpr int STAGE = 2 * HALF;
  static constexpr int S = 196608 / (W * STAGE);    // stages per warp
  static constexpr int BLOCK = 16 * W;              // tokens
  static constexpr int RING = W * S * STAGE;
  static constexpr int JOIN = RING;                 // 8 rows of every warp's sums
  static constexpr int ML = JOIN + W * 8 * DP * 4;  // [W][16][2] every warp's max and sum per row
  static constexpr int PRE = ML + W * 128;          // [128] blocks per item before each group of sequences
  static constexpr int MISC = PRE + 512;            // [8] scan scratch
  static constexpr int SMEM = MISC + 32;
  static_assert(SMEM <= 232448, "a CTA's shared memory");
};

struct DecodeArgs {
  const void* q;
  void* out;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t* tables;
  const int32_t* lens;
  float* part;      // two for each CTA: [slots][prows][DP] sums, then [slots][prows][2] (max, sum)
  uint32_t* count;  // kCounterBytes
  int64_t slots;
  int prows;        // rows of a partial: 8 or 16
  int64_t q_row, q_head, o_row, o_head, table_row;
  int64_t room;     // tokens a table row has room for
  int batch, hkv, group, hblocks, d, page_size, num_pages, window;
  float s2;         // scale * log2(e)
};

// The work list cut into runs, the first `extra` of them one block longer than `size`. (The
// host refuses lists of 2^31 blocks and more.)
struct Runs {
  int size, extra;
  __device__ __forceinline__ int begin(int r) const { return r * size + min(r, extra); }
  __device__ __forceinline__ int holding(int block) const {  // the run of a block
    const int longer = extra * (size + 1);
    return block < longer ? block / (size + 1) : extra + (block - longer) / size;
  }
};

// A walk over the blocks of a run: where the current item's blocks lie. An item has nb blocks
// of tokens, then one that stands for its own cost.
struct Walk {
  int left, base;        // blocks of the run to come, first block of the current sequence
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
  w.k0 += w.n;
  for (;;) {
    if (w.left <= 0) return false;
    if (w.k0 < w.nb) break;
    // past the item's last block
    if (w.nb > 0) --w.left;
    w.k0 = 0;
    if (w.nb == 0 || ++w.item >= hi) {
      w.item = 0;
      w.base += (w.nb ? w.nb + 1 : 0) * hi;
      if (++w.b >= a.batch) {  // the end, or the lengths changed under the kernel
        w.left = 0;
        return false;
      }
      walk_load<BLOCK>(a, w);
    }
  }
  w.n = min(w.nb - w.k0, w.left);
  w.starts = w.k0 == 0;
  w.ends = w.k0 + w.n == w.nb;
  w.left -= w.n;
  return true;
}

// To block 0 of run r: the group of sequences that holds it, by all lanes of a warp.
template <int BLOCK>
__device__ __forceinline__ void walk_to(const DecodeArgs& a, Walk& w, const Runs& runs, int r, const int* pre, int gs,
                                        int hi, int lane) {
  const int u = runs.begin(r);
  w.left = runs.begin(r + 1) - u;
  int g = -1;
#pragma unroll
  for (int x = 0; x < 4; ++x) g += __popc(__ballot_sync(0xFFFFFFFFu, pre[x * 32 + lane] * hi <= u));
  g = max(g, 0);
  w.b = min(g * gs, a.batch - 1);
  w.base = pre[g] * hi;
  walk_load<BLOCK>(a, w);
  while (w.b + 1 < a.batch && (w.nb == 0 || u >= w.base + (w.nb + 1) * hi)) {
    w.base += (w.nb ? w.nb + 1 : 0) * hi;
    ++w.b;
    walk_load<BLOCK>(a, w);
  }
  w.item = (u - w.base) / (w.nb + 1);
  w.k0 = u - w.base - w.item * (w.nb + 1);
  w.n = 0;  // the first segment starts here
}

// 16 bytes to shared memory, the first `bytes` (0 or 16) of them from p, the rest zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* p, uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(p), "r"(bytes), "l"(policy)
               : "memory");
}

__device__ __forceinline__ uint32_t arrive_acq_rel(uint32_t* p) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}

template <int DP, int DT>
__global__ void __launch_bounds__(Shape<DP>::W * 32, 1) paged_decode_kernel(const __grid_constant__ DecodeArgs a) {
  using C = Shape<DP>;
  constexpr int W = C::W, S = C::S, BLOCK = C::BLOCK, T = W * 32;
  // a stage: K, then V, 16 tokens each: row r, 128-byte column block c at (r / 8) * 1024 +
  // c * 2048 + (r % 8) * 128, its 16-byte chunks in the order chunk ^ (r % 8)
  constexpr int HS = 1024, BS = 2048;
  // 16-bit floats underflow early (2^-24), and a long tail of small weights can add up: theirs
  // are kept 2^14 larger, the sum too
  constexpr float kUp = DT == GGUFMM_F16 ? 14.f : 0.f;
  extern __shared__ __align__(1024) uint8_t ring[];
  float* join = reinterpret_cast<float*>(ring + C::JOIN);
  float* ml = reinterpret_cast<float*>(ring + C::ML);
  int* pre = reinterpret_cast<int*>(ring + C::PRE);
  int* misc = reinterpret_cast<int*>(ring + C::MISC);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* mine = ring + warp * S * C::STAGE;
  pdl_wait();
  pdl_trigger();

  // ---- the work: blocks per item before each of 128 groups of sequences ----------------
  const int hi = a.hkv * a.hblocks;  // items per sequence
  const int gs = (a.batch + 127) / 128;
  int mine_b = 0, inc;
  if (tid < 128) {
    for (int b = tid * gs; b < min((tid + 1) * gs, a.batch); ++b) {
      int lo;
      bool cut;
      const int len = seq_len(a, b, &cut);
      if (cut && blockIdx.x == 0) atomicOr(&g_device_error, kErrIndex);
      const int nb = seq_blocks<BLOCK>(a, len, &lo);
      mine_b += nb ? nb + 1 : 0;
    }
    inc = mine_b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) misc[warp] = inc;
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (tid < 128 && i == warp) pre[tid] = total + inc - mine_b;
    total += misc[i];
  }
  __syncthreads();
  const int blocks = total * hi;
  const int me = static_cast<int>(blockIdx.x);
  const int nruns = min(static_cast<int>(gridDim.x), blocks);
  Runs runs;
  runs.size = nruns ? blocks / nruns : 0;
  runs.extra = blocks - runs.size * nruns;
  // sequences that see nothing: zeros
  for (int b = me; b < a.batch; b += gridDim.x) {
    int lo;
    bool cut;
    if (seq_blocks<BLOCK>(a, seq_len(a, b, &cut), &lo)) continue;
    const int per = a.d / 8, heads = a.hkv * a.group;
    for (int i = tid; i < heads * per; i += T)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + b * a.o_row + i / per * a.o_head + i % per * 8) =
          make_uint4(0, 0, 0, 0);
  }
  if (me >= nruns) return;
  Walk cw;
  walk_to<BLOCK>(a, cw, runs, me, pre, gs, hi, lane);
  // ---- the producer half of each warp: the chunks of its walk, S stages ahead ---------------
  Walk pw = cw;
  const uint64_t policy = l2_evict_first_policy();
  int pk = 0, pn = 0, pbase = 0;  // next block of the segment, their number, block of pid's lane 0
  int pid0 = 0, pid1 = 0;         // lane i: pages of the chunk's first and second 8 tokens, block pbase + i,
  int off0 = 0, off1 = 0;         // and their slots there; a negative page is not read
  int stage_p = 0;
  auto load_pages = [&]() {
    pbase = pk;
    const int t = (pw.f + pw.k0 + pk + lane) * BLOCK + warp * 16;
    const int32_t* row = a.tables + pw.b * a.table_row;
    auto page_of = [&](int tok, int* off) {
      if (tok >= pw.len || tok + 8 <= pw.lo) return -1;
      const int at = tok / a.page_size, p = row[at];
      *off = tok - at * a.page_size;
      if (p >= 0 && p < a.num_pages) return p;
      atomicOr(&g_device_error, kErrIndex);
      return -1;
    };
    if (pk + lane < pn) {
      pid0 = page_of(t, &off0);
      pid1 = page_of(t + 8, &off1);
    }
  };
  // a lane copies chunk lane % CH of a row, RPI rows of the warp at a time; columns past the
  // head's are zeros
  constexpr int CH = DP / 8, RPI = 32 / CH, NSWZ = 8 / RPI;
  const int ch = lane % CH, sub = lane / CH;
  const bool col = ch * 8 < a.d;
  const uint32_t bytes_l = col ? 16 : 0;
  const int64_t lane_k = sub * a.k_slot + (col ? ch * 8 : 0), lane_v = sub * a.v_slot + (col ? ch * 8 : 0);
  const int64_t k_step = RPI * a.k_slot, v_step = RPI * a.v_slot;
  const uint16_t* k_l = a.k;  // of the segment's head
  const uint16_t* v_l = a.v;
  const uint32_t mine_u = smem_u32(mine), dst_l = mine_u + (ch >> 3) * BS + sub * 128;
  uint32_t swz[NSWZ];  // of rows x + sub
#pragma unroll
  for (int x = 0; x < NSWZ; ++x) swz[x] = ((ch & 7) ^ (x * RPI + sub)) << 4;
  auto produce = [&]() {  // the next chunk of this warp into its next stage, if there is one
    for (;;) {
      if (pk >= pn) {
        if (!walk_next<BLOCK>(a, pw, hi)) break;
        pk = 0;
        pn = pw.n;
        load_pages();
        const int head = pw.item / a.hblocks;
        k_l = a.k + head * a.k_head + lane_k;
        v_l = a.v + head * a.v_head + lane_v;
      } else if (pk - pbase == 32) {
        load_pages();
      }
      const int t = (pw.f + pw.k0 + pk) * BLOCK + warp * 16;
      const int sel = pk - pbase;
      ++pk;
      if (t >= pw.len || t + 16 <= pw.lo) continue;
      const uint32_t dst = dst_l + stage_p * C::STAGE;
      const bool inside = t >= pw.lo && t + 16 <= pw.len;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int page = __shfl_sync(0xFFFFFFFFu, h ? pid1 : pid0, sel), off = __shfl_sync(0xFFFFFFFFu, h ? off1 : off0, sel);
        if (inside && page >= 0) {
          const uint16_t* ks = k_l + page * a.k_page + off * a.k_slot;
          const uint16_t* vs = v_l + page * a.v_page + off * a.v_slot;
#pragma unroll
          for (int x = 0; x < 8; x += RPI) {
            const uint32_t at = dst + h * HS + x * 128 + swz[x / RPI % NSWZ];
            copy16(at, ks, bytes_l, policy);
            copy16(at + C::HALF, vs, bytes_l, policy);
            ks += k_step;
            vs += v_step;
          }
        } else {
          // tokens that are not seen are zeros: what lies there may be anything, NaN too, and a
          // weight of 0 must meet 0
#pragma unroll
          for (int x = 0; x < 8; x += RPI) {
            const int tok = t + h * 8 + x + sub;
            const bool in = page >= 0 && tok >= pw.lo && tok < pw.len;
            const int64_t pg = in ? page : 0, of = in ? off + x : 0;
            const uint32_t at = dst + h * HS + x * 128 + swz[x / RPI % NSWZ];
            copy16(at, in ? k_l + pg * a.k_page + of * a.k_slot : a.k, in ? bytes_l : 0, policy);
            copy16(at + C::HALF, in ? v_l + pg * a.v_page + of * a.v_slot : a.v, in ? bytes_l : 0, policy);
          }
        }
      }
      stage_p = stage_p + 1 == S ? 0 : stage_p + 1;
      break;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // one group a call, empty at the end
  };
#pragma unroll 1
  for (int i = 0; i < S; ++i) produce();

  // ---- the consumer half -------------------------------------------------------------
  const int g = lane >> 2, t4 = lane & 3;
  int stage_c = 0;
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
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
      __syncwarp();
      {
        const bool edge = t < cw.lo || t + 16 > cw.len;
        // scores: 16 query heads x 16 tokens
        float s[2][4] = {}, s_odd[2][4] = {};  // even and odd steps apart: half as long a chain
#pragma unroll
        for (int k16 = 0; k16 < DP / 16; ++k16) {
          // matrices: tokens 0-7 / 8-15 x columns k16*16 + 0-7 / 8-15
          const int c = k16 * 2 + (lq & 1), cc = c & 7;
          uint32_t b[4];
          ldsm4(kb + (lq >> 1) * HS + (c >> 3) * BS + lr * 128 + ((cc ^ lr) << 4), b);
          mma_16816<DT>(k16 & 1 ? s_odd[0] : s[0], qf[k16], b[0], b[1]);
          mma_16816<DT>(k16 & 1 ? s_odd[1] : s[1], qf[k16], b[2], b[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[n][i] = (s[n][i] + s_odd[n][i]) * a.s2;
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
        const float z0 = (m0 == -INFINITY ? 0.f : m0) - kUp, z1 = (m1 == -INFINITY ? 0.f : m1) - kUp;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n][0] = exp2_fast(s[n][0] - z0);
          s[n][1] = exp2_fast(s[n][1] - z0);
          s[n][2] = exp2_fast(s[n][2] - z1);
          s[n][3] = exp2_fast(s[n][3] - z1);
          l0 += s[n][0] + s[n][1];
          l1 += s[n][2] + s[n][3];
        }
        // the weights, at most 1 (2^kUp), rounded to the cache's type for the product with v, whose
        // two operands have one type: a relative 2^-9 (f16 2^-12) each and half as much on average,
        // as the output's own rounding; their sum is not rounded. Relative error of the output against
        // 64 bits 0.0017 to 0.0018 where 32-bit weights give 0.0016 to 0.0017 (f16 0.00022 and 0.00020)
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
      produce();
    }
    // ---- join the warps --------------------------------------------------------------
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);
    if (t4 == 0) {
      *reinterpret_cast<float2*>(ml + (warp * 16 + g) * 2) = make_float2(m0, l0);
      *reinterpret_cast<float2*>(ml + (warp * 16 + g + 8) * 2) = make_float2(m1, l1);
    }
    const bool whole = cw.starts && cw.ends;
    const int item0 = cw.base + cw.item * (cw.nb + 1);  // first block of the item
    // a run has at most one piece of an item begun before it, and one of an item that goes on after it
    const int slot = me * 2 + (cw.starts ? 1 : 0);
    float* const part_ml = a.part + a.slots * a.prows * DP;
    uint16_t* outp = static_cast<uint16_t*>(a.out) + cw.b * a.o_row + qh0 * a.o_head;
#pragma unroll 1
    for (int h = 0; h * 8 < rows; ++h) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2*>(join + (warp * 8 + g) * DP + i * 8 + t4 * 2) =
            make_float2(h ? o[i][2] : o[i][0], h ? o[i][3] : o[i][1]);
      __syncthreads();
      for (int e = tid; e < 8 * DP / 4; e += T) {
        const int r = e / (DP / 4), c = e % (DP / 4) * 4, row = h * 8 + r;
        if (row >= rows) continue;
        float2 w[W];
        float mr = -INFINITY;
#pragma unroll
        for (int x = 0; x < W; ++x) {
          w[x] = *reinterpret_cast<const float2*>(ml + (x * 16 + row) * 2);
          mr = fmaxf(mr, w[x].x);
        }
        const float zr = mr == -INFINITY ? 0.f : mr;
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < W; ++x) {
          const float f = exp2_fast(w[x].x - zr);
          const float4 v = *reinterpret_cast<const float4*>(join + (x * 8 + r) * DP + c);
          l += w[x].y * f;
          acc.x += v.x * f;
          acc.y += v.y * f;
          acc.z += v.z * f;
          acc.w += v.w * f;
        }
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          if (c < a.d)
            *reinterpret_cast<uint2*>(outp + row * a.o_head + c) =
                make_uint2(pack16<DT>(acc.x * inv, acc.y * inv), pack16<DT>(acc.z * inv, acc.w * inv));
        } else {
          __stcg(reinterpret_cast<float4*>(a.part + (static_cast<int64_t>(slot) * a.prows + row) * DP + c), acc);
          if (c == 0) __stcg(reinterpret_cast<float2*>(part_ml + (static_cast<int64_t>(slot) * a.prows + row) * 2), make_float2(mr, l));
        }
      }
      __syncthreads();
    }
    if (whole) continue;
    // ---- join the CTAs of this item: the last one to arrive adds the partials ---------------
    const int c0 = cw.starts ? me : runs.holding(item0), c1 = cw.ends ? me : runs.holding(item0 + cw.nb - 1);
    if (tid == 0) misc[7] = arrive_acq_rel(a.count + c0) + 1 == static_cast<uint32_t>(c1 - c0 + 1);
    __syncthreads();
    const bool last = misc[7] != 0;
    __syncthreads();  // misc[7] is written again at the next item
    if (!last) continue;
    if (tid == 0) a.count[c0] = 0;
    for (int e = tid; e < rows * (DP / 4); e += T) {
      const int row = e / (DP / 4), c = e % (DP / 4) * 4;
      float mr = -INFINITY, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      constexpr int K = 8;  // partials under way at a time
      for (int k = c0; k <= c1; k += K) {
        float2 w[K];
        float4 v[K];
        float mk = mr;
#pragma unroll
        for (int x = 0; x < K; ++x) {
          const int64_t at = (2 * static_cast<int64_t>(k + x) + (k + x == c0)) * a.prows + row;
          w[x] = k + x <= c1 ? __ldcg(reinterpret_cast<const float2*>(part_ml + at * 2)) : make_float2(-INFINITY, 0.f);
          v[x] = k + x <= c1 ? __ldcg(reinterpret_cast<const float4*>(a.part + at * DP + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int x = 0; x < K; ++x) mk = fmaxf(mk, w[x].x);
        const float z = mk == -INFINITY ? 0.f : mk, f0 = exp2_fast(mr - z);
        l *= f0;
        acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
        for (int x = 0; x < K; ++x) {
          const float f = exp2_fast(w[x].x - z);
          l += w[x].y * f;
          acc.x += v[x].x * f;
          acc.y += v[x].y * f;
          acc.z += v[x].z * f;
          acc.w += v[x].w * f;
        }
        mr = mk;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (c < a.d)
        *reinterpret_cast<uint2*>(outp + row * a.o_head + c) =
            make_uint2(pack16<DT>(acc.x * inv, acc.y * inv), pack16<DT>(acc.z * inv, acc.w * inv));
    }
  }
}

template <int DP, int DT>
cudaError_t launch(const DecodeArgs& a, int grid, int dev, cudaStream_t st) {
  auto fn = paged_decode_kernel<DP, DT>;
  static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
  if (!(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::SMEM);
    if (e != cudaSuccess) return e;
    ready.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_release);
  }
  return pdl_launch(fn, dim3(static_cast<unsigned>(grid)), dim3(Shape<DP>::W * 32), Shape<DP>::SMEM, st, a);
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

}  // namespace

size_t paged_decode_workspace(int64_t group, int64_t head_dim) {
  return kCounterBytes + static_cast<size_t>(2 * kMaxGrid) * (group <= 8 ? 8 : 16) * (padded_dim(head_dim) + 2) * 4;
}

cudaError_t launch_paged_decode(const ggufmm_attention_args& p, void* workspace, cudaStream_t st) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int grid = std::min(std::max(device_info(dev).sms, 1), kMaxGrid);
  DecodeArgs a;
  a.q = p.q;
  a.out = p.out;
  a.k = static_cast<const uint16_t*>(p.k);
  a.v = static_cast<const uint16_t*>(p.v);
  a.k_page = p.k_page;
  a.k_head = p.k_head;
  a.k_slot = p.k_slot;
  a.v_page = p.v_page;
  a.v_head = p.v_head;
  a.v_slot = p.v_slot;
  a.tables = static_cast<const int32_t*>(p.tables);
  a.lens = static_cast<const int32_t*>(p.lens);
  a.count = static_cast<uint32_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  a.slots = static_cast<int64_t>(2) * kMaxGrid;
  a.prows = p.q_heads / p.kv_heads <= 8 ? 8 : 16;
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
  a.s2 = static_cast<float>(p.scale * 1.4426950408889634);
  const bool f16 = p.dtype == GGUFMM_F16;
  switch (padded_dim(p.head_dim)) {
    case 64: return f16 ? launch<64, GGUFMM_F16>(a, grid, dev, st) : launch<64, GGUFMM_BF16>(a, grid, dev, st);
    case 128: return f16 ? launch<128, GGUFMM_F16>(a, grid, dev, st) : launch<128, GGUFMM_BF16>(a, grid, dev, st);
    default: return f16 ? launch<256, GGUFMM_F16>(a, grid, dev, st) : launch<256, GGUFMM_BF16>(a, grid, dev, st);
  }
}

cudaError_t attn_decode_device_error(int* v, int clear, cudaStream_t st) { return tu_device_error(v, clear, st); }

}  // namespace ggufmm
