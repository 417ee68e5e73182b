// bfloat16 attention of a few new tokens a sequence over a cache held in 8 or 4 bits (formats: top of
// kv_quant.cu): single tokens of a decode step, with their rotary encoding and cache write inside, and
// short runs of tokens already stored.  head_dim 64 or 128, any group size, pages of a multiple of 64.
//
// Mathematics.  The codes go through the integer tensor cores as they are; scales enter outside:
//   8 bits  s_j = sk_j (q . ck_j),                            out = sum_j (p_j sv_j) cv_j / sum_j p_j
//   4 bits  s_j = sum_g sk_jg (q_g . (ck_jg - 8)) + mk_jg sum(q_g),
//           out_g = (sum_j (p_j sv_jg) cv_jg + sum_j p_j (mv_jg - 8 sv_jg)) / sum_j p_j
// A query row becomes whole numbers of 16 bits in both formats (largest element 32512: a step is 1 / 32512 of it, also
// for the small elements of a row in which one stands out, where bfloat16 would keep 8 bits of each), split into two
// bytes that take two columns of the product; the integer scores are exact.  For the value product the p_j sv_j of one
// step of keys become whole numbers of 16 bits too, against the largest of the step, again two bytes in two columns:
// within a step 2^-17 of the largest is lost (the sum of p, and in 4 bits the mids' share, take p unrounded), and a
// step's integer sum goes into the 32-bit accumulators with the step's own factor, so nothing is lost between steps.
// Statistics and sums are 32 bits.
//
// Shape.  The products are taken transposed, keys (then value dims) on the MMA's 16 rows and the query
// rows on its columns, four of them (times two bytes) a tile of eight: with four query heads to a
// kv head no column is empty, an accumulator pair is one score, and P moves from one product to the
// other by a byte permutation and a movmatrix.  Codes need no conversion: a key's row is the operand
// (4 bits: an AND or a shift and an AND for four codes), values are brought to four keys a
// register by two byte permutations for eight codes.  (Tried first: codes converted to float16 for
// m16n8k16 products, 490 instructions for 32 keys of 8 bits, 850 for 32 of 4 bits, bound by issue and
// latency: 64 sequences of up to 4,500 keys 101 us, of 9,000 in 4 bits 194 us.)  What should bound it is
// memory: a key and value of a head are 264 bytes (8 bits, head_dim 128) or 144 (4 bits).
//
// Work is cut evenly: all (sequence, kv head) units' key tiles stand in one row that is shared out over two or
// three blocks an SM, so unequal lengths leave no tail; a warp's loads (TMA, its own ring of stages, the scales
// along with the codes) run on across the border between two units.  Where every unit can have blocks of its own for
// at most two steps more a block, it gets them: a border costs about that much.  A unit that was cut is joined
// in block order by the block that finishes it last.
//
// Measured from a graph (keys and values at the measured copy rate in brackets; calls one by one take 2 to 8 % more): 64
// sequences of up to 4,500 keys, 8 bits, 32 heads on 8, 80 us (71); 64 of up to 9,000 in 4 bits 96 (77); one of 130,018
// in 8 bits 50 (42); one of 34 keys 6.2, the latency of the chain batch -> block table -> keys -> softmax -> values.  Three
// blocks an SM for 8 bits 82 us, rings of four stages there 83.  4 bits are bound by issue: 0.47 instructions a cycle and
// scheduler with two warps on it, 47 million of them for the 64 sequences (8 bits: 0.29).
// More rows a kv head repeat products and softmax for every tile of four: 64 sequences of up to 4,500 with groups of 8 take
// 87 us (8 bits; 71) and 82 (4 bits; 39), 32 of them with groups of 16 71 (36) and 89 (20); 4 new tokens on 6 of up to 16,000 47
// (18.6) and 55 (10.2).  The instances of 8 and 16 rows at 128 dims use all 255 registers and spill (bytes stored / loaded:
// 8 bits, 16 rows 48 / 36; 4 bits, 8 rows 56 / 52, 16 rows 280 / 224), outside the steps: 0.1 and 0.2 % of the instructions.  64 dims take a step's fixed work for half the bytes: two of
// 60,001 in 4 bits 23 (10), in 8 bits 29 (19).
#include "attention_mma.cuh"
#include "kv_quant.cuh"
#include "load_ring.h"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

#include <type_traits>

namespace siar {

struct QuantAttnParams {
  const __nv_bfloat16* qkv;      // [N, (Hq + 2 Hkv) D]
  const __half* q16;             // or queries as float16 [N, Hq, D] times a power of two a row, q_factor [N, Hq]
  const float* q_factor;
  uint8_t* k_pool;
  uint8_t* v_pool;
  void* k_scale;
  void* v_scale;
  const int* block_table;
  const int* slot_ids;
  const int* q_start;
  const int* base_len;
  const float* inv_freq;         // fused rotation of the new token, or nullptr
  __nv_bfloat16* out;            // [N, Hq D]
  float* scratch;                // [blocks][2] segments of cut units
  int* counters;                 // [units], zero between launches
  int* status;
  int B, Hq, Hkv, page_tokens, max_pages, n_pages;
  int page_shift;                // log2(page_tokens), or -1
  int fused;                     // rotate and (write_kv) store the new token here; one token a sequence
  int write_kv;
  int most_new;                  // sequences with more new tokens than this are left to another kernel
  float sl2;                     // scale * log2(e)
};

template <int BITS, int D, int NT>
struct QuantAttn {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kWarpKeys = D == 128 && (BITS == 8 || NT == 4) ? 32 : 64;     // keys per warp and step
  static constexpr int kBlockKeys = 4 * kWarpKeys;
  static constexpr int kTileBytes = kWarpKeys * kRowBytes;
  static constexpr int kGroups = BITS == 8 ? 1 : D / kQuantGroup;
  static constexpr int kScaleBytes = kWarpKeys * 4 * kGroups;        // float32, or (scale, mid) bfloat16 per run
  // blocks an SM and pipeline depth: what shared memory (and, for many rows, registers) leave room for
  static constexpr int kBlocksPerSM = NT == 1 && D == 64 ? 3 : 2;
  static constexpr int kStages = kTileBytes < 4096 && NT > 1 ? 4 : 2;
  static constexpr int kRows = 4 * NT;                               // query rows of a unit
  static constexpr int kMT = D / 16;                                 // row tiles of the value product
  static constexpr int kQStride = D + 16;                            // bytes per column of query bytes in shared memory
  static constexpr int kRegs = kMT * NT * 2;                         // accumulators of a lane
  // shared memory
  static constexpr int kTiles = 0;                                   // [stages][warp][K | V]
  static constexpr int kScales = kTiles + kStages * 4 * 2 * kTileBytes;
  static constexpr int kJoin = kScales + kStages * 4 * 2 * kScaleBytes;   // [2][kRegs][32] floats
  static constexpr int kQ = kJoin + 2 * kRegs * 32 * 4;
  static constexpr int kSmem = kQ + 8 * NT * kQStride;
  static constexpr int kSegFloats = (kRegs + 2 * NT) * 32;           // accumulators, references, sums
  // an SM has 228 KB, of which every block takes 1 KB, its static arrays (under 4.2 KB) and what aligns the tiles
  static_assert(kBlocksPerSM * (kSmem + 1024 + 1024 + (NT == 1 ? 1500 : NT == 2 ? 2100 : 3300)) <= 228 * 1024, "blocks an SM");
};
constexpr float kFixedP = 65500.f;                // p sv of a step's largest term, as a whole number
constexpr float kFixedQ = 32512.f;                // a query row's largest element, as a whole number: 127 x 256

// D (int32) = C + A B for bytes; ASIGN / BSIGN: signed operands, FIRST: C is zero.
template <bool ASIGN, bool BSIGN, bool FIRST>
__device__ __forceinline__ void mma_bytes(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define SIAR_MMA(AT, BT)                                                                                                    \
  if (FIRST)                                                                                                                \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." AT "." BT ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};" \
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                            \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));                                            \
  else                                                                                                                      \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." AT "." BT ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"     \
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                            \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if (ASIGN && BSIGN) { SIAR_MMA("s8", "s8"); }
  else if (ASIGN) { SIAR_MMA("s8", "u8"); }
  else if (BSIGN) { SIAR_MMA("u8", "s8"); }
  else { SIAR_MMA("u8", "u8"); }
#undef SIAR_MMA
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// Where byte `off` of a tile stands: the TMA swizzle whose span is the row (128, 64 or 32 bytes).
template <int ROW>
__device__ __forceinline__ uint32_t swizzled(uint32_t off) {
  return off ^ (((off >> 7) & (ROW / 16 - 1)) << 4);
}

// ceil(steps / chunk) for steps below 2^24: the float quotient is off by at most one.
__device__ __forceinline__ int chunks_of(int steps, int chunk) {
  int q = (int)__fdividef((float)(steps + chunk - 1), (float)chunk);
  q -= q * chunk > steps + chunk - 1;
  return q + ((q + 1) * chunk <= steps + chunk - 1);
}

// One sequence's units: (row tile, kv head), all of T block steps.
struct QuantSeq {
  int b, base, t0, q_len, slot, len, T, row_tiles;
};

template <int BITS, int D, int NT>
__global__ void __launch_bounds__(128, (QuantAttn<BITS, D, NT>::kBlocksPerSM))
attn_quant_kernel(const __grid_constant__ QuantAttnParams P, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map) {
  using C = QuantAttn<BITS, D, NT>;
  constexpr int WK = C::kWarpKeys, KT = WK / 16, RB = C::kRowBytes, NG = C::kGroups, MT = C::kMT;
  pdl_launch_dependents();
  extern __shared__ unsigned char smem_base[];
  unsigned char* smem = smem_base + ((1024 - (smem_u32(smem_base) & 1023)) & 1023);     // the swizzle pattern's period
  __shared__ __align__(8) uint64_t bars[4][C::kStages];
  __shared__ float cs_s[D];                       // cosines, sines of the new token's position
  __shared__ __align__(16) uint32_t new_codes[2][RB / 4];     // the new token's key and value,
  __shared__ uint32_t new_scale[2][NG];                       // codes and scales
  __shared__ float f_s[C::kRows];
  __shared__ int qsum_s[C::kRows][NG];
  __shared__ float ml_s[2][NT * 2][32];
  __shared__ int last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  float freq = 0.f;                               // a constant of the model, so it may be read in front of the wait
  if (P.fused && P.inv_freq != nullptr && threadIdx.x < D / 2) freq = P.inv_freq[threadIdx.x];
  pdl_wait();
  asm volatile("fence.proxy.async.global;" ::: "memory");      // rows that the kernel in front stored, for the TMA

  const int G = P.Hq / P.Hkv;
  const int cap = P.max_pages * P.page_tokens;
  bool past_table = false;                        // a token behind what a row of the block table names
  auto load_seq = [&](int b) {
    QuantSeq s;
    s.b = b;
    s.base = P.base_len[b];
    s.t0 = P.q_start[b];
    s.q_len = P.q_start[b + 1] - s.t0;
    s.slot = P.slot_ids[b];
    s.len = min(s.base + s.q_len, cap);
    past_table |= s.base + s.q_len > cap;
    s.T = max(0, (s.len + C::kBlockKeys - 1) / C::kBlockKeys);
    s.row_tiles = s.q_len <= P.most_new ? max(0, (s.q_len * G + C::kRows - 1) / C::kRows) : 0;
    return s;
  };
  // ---- this block's share of all block steps
  // Sums over all sequences, 32 a time (a lane keeps its first one); a sum of 2^26 or more is refused, so a lane's
  // part may stop there.
  QuantSeq own = {};
  if (lane < P.B) own = load_seq(lane);
  auto total_of = [&](auto weight) {
    long long mine = weight(own);
    for (int b = lane + 32; b < P.B; b += 32) mine += weight(load_seq(b));
    return __reduce_add_sync(0xffffffffu, (unsigned)min(mine, 1ll << 26));
  };
  const unsigned sum = total_of([&](const QuantSeq& s) { return (long long)s.T * (s.row_tiles * P.Hkv); });
  if (sum >= 1u << 26) {
    if (threadIdx.x == 0) atomicOr(P.status, kStatusLengthPastGrid);
    return;
  }
  const int total = (int)sum;
  const unsigned units = total_of([&](const QuantSeq& s) { return s.T > 0 ? (long long)(s.row_tiles * P.Hkv) : 0ll; });
  // at least one step a block: a block without one would be waited for by the join of a unit around it
  int nb = min((int)gridDim.x, total);
  if ((int)blockIdx.x >= nb) return;
  const int each = total / nb, odd = total % nb;  // the first `odd` blocks take one step more
  // Where it costs a block at most kCrossing steps more than an even share, no block meets two units: every unit
  // gets ceil(T / chunk) blocks (a border between two units costs a block about that many steps: a join of its
  // warps, a partial result, the next query).
  constexpr int kCrossing = 2;
  int chunk = each + (odd > 0);
  bool by_unit = false;
  for (const int most = chunk + kCrossing; chunk <= most && units <= gridDim.x; ++chunk) {
    const unsigned need = total_of([&](const QuantSeq& s) { return (long long)chunks_of(s.T, chunk) * (s.row_tiles * P.Hkv); });
    by_unit = need <= gridDim.x;
    if (by_unit) {
      nb = (int)need;
      break;
    }
  }
  if ((int)blockIdx.x >= nb) return;
  auto parts_of = [&](const QuantSeq& s) { return by_unit ? chunks_of(s.T, chunk) : s.T; };   // blocks, or steps, of a unit
  auto begin_of = [&](int i) { return i * each + min(i, odd); };
  auto block_of = [&](int step) { return step < odd * (each + 1) ? step / (each + 1) : odd + (step - odd * (each + 1)) / each; };
  const int start = by_unit ? blockIdx.x : begin_of(blockIdx.x);
  QuantSeq cu;                                    // unit that is computed: sequence, row tile, kv head, step
  int c_rt, c_kvh, c_t, n_steps;
  int unit_begin, begin, end;                     // the current unit's first step and the block's steps, in one row of all steps
  int part = 0;                                   // by_unit: the block's place among its unit's blocks
  {
    int before = 0, b0 = 0;
    while (true) {                                // 32 sequences at a time
      int mine = 0;
      if (b0 + lane < P.B) {
        const QuantSeq s = b0 == 0 ? own : load_seq(b0 + lane);
        mine = parts_of(s) * s.row_tiles * P.Hkv;
      }
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + incl > start);
      if (past != 0 || b0 + 32 >= P.B) {
        const int at = past != 0 ? __ffs(past) - 1 : 31;
        before += __shfl_sync(0xffffffffu, incl - mine, at);
        cu = load_seq(min(b0 + at, P.B - 1));
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      b0 += 32;
    }
    const int parts = parts_of(cu), in_seq = start - before, unit = in_seq / parts;
    part = in_seq % parts;
    c_rt = unit / P.Hkv;
    c_kvh = unit % P.Hkv;
    if (by_unit) {                                // the unit's steps shared out evenly over its blocks
      const int per = cu.T / parts, more = cu.T % parts;
      unit_begin = 0;
      begin = part * per + min(part, more);
      end = begin + per + (part < more);
      c_t = begin;
    } else {
      begin = start;
      end = begin_of(blockIdx.x + 1);
      c_t = part;
      unit_begin = begin - c_t;
    }
    n_steps = end - begin;
  }
  auto page_index = [&](int pos) { return P.page_shift >= 0 ? pos >> P.page_shift : pos / P.page_tokens; };

  // ---- the unit's query rows (a warp takes rows warp, warp + 4, ...; a lane dims lane + 32 i) and, where the
  // unit's last step falls into this block, the new token's key (warp 0) and value (warp 1).  They are asked for
  // ahead of the block's first tiles, and ahead of the join in front of a later unit.
  const size_t qkv_row = (size_t)(P.Hq + 2 * P.Hkv) * D;
  float qa[NT][D / 32], ta[D / 32];
  int t_page = -1;                                // the page of the new token
  auto has_new = [&](const QuantSeq& s, int t, int left) {       // left: steps of the block from t on
    return P.fused && P.write_kv && s.base < cap && s.base / C::kBlockKeys >= t && s.base / C::kBlockKeys < t + left;
  };
  auto fetch = [&](const QuantSeq& s, int rt, int kvh, int t, int left) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int row = rt * C::kRows + 4 * j + warp;
      const bool in = row < s.q_len * G;
      const int token = s.t0 + (in ? row / G : 0), head = kvh * G + (in ? row % G : 0);
      if (P.q16 != nullptr) {
        const __half* src = P.q16 + ((size_t)token * P.Hq + head) * D + lane;
        const float f = P.q_factor[(size_t)token * P.Hq + head];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) qa[j][i] = in ? __half2float(src[32 * i]) * f : 0.f;
      } else {
        const __nv_bfloat16* src = P.qkv + (size_t)token * qkv_row + (size_t)head * D + lane;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) qa[j][i] = in ? __bfloat162float(src[32 * i]) : 0.f;
      }
    }
    if (warp < 2 && has_new(s, t, left)) {
      const __nv_bfloat16* src = P.qkv + (size_t)s.t0 * qkv_row + (size_t)(P.Hq + warp * P.Hkv + kvh) * D + lane;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) ta[i] = __bfloat162float(src[32 * i]);
      t_page = P.block_table[(size_t)s.slot * P.max_pages + page_index(s.base)];
    }
  };

  // ---- this warp's loads: the same walk, ahead of the computation
  QuantSeq lu = cu;
  int l_rt = c_rt, l_kvh = c_kvh, l_t = c_t, l_left = n_steps;
  LoadRing<C::kStages> ring;
  // the same answer in every lane: what follows is work of the whole warp
  auto arrived = [&](int stage, int parity) { return __all_sync(0xffffffffu, mbar_wait(&bars[warp][stage], parity)) != 0; };
  bool absent_page = false;
  auto next_seq = [&](const QuantSeq& s) {        // the next sequence that has steps (there is one)
    int b = s.b + 1;
    QuantSeq n = load_seq(b);
    while (n.T * n.row_tiles == 0) n = load_seq(++b);
    return n;
  };
  // Lane i holds the page of the warp's tile i steps on from l_page0 in the load cursor's unit; asked for ahead
  // of its use, 32 steps at a time.
  int l_page0 = 0, l_pages = 0;
  auto ask_pages = [&]() {
    const int w0 = (l_t + lane) * C::kBlockKeys + warp * WK;
    l_page0 = l_t;
    l_pages = l_left > 0 && w0 < lu.len ? P.block_table[(size_t)lu.slot * P.max_pages + page_index(w0)] : 0;
  };
  ask_pages();
  fetch(cu, c_rt, c_kvh, c_t, n_steps);
  auto issue_next = [&]() {
    while (l_left > 0 && ring.room()) {
      const int w0 = l_t * C::kBlockKeys + warp * WK;
      const bool has = w0 < lu.len;
      if (has) {
        int page = __shfl_sync(0xffffffffu, l_pages, l_t - l_page0);
        if (page < 0 || page >= P.n_pages) { absent_page = true; page = 0; }
        const int s = ring.next();
        if (lane == 0) {
          const int row = (page * P.Hkv + l_kvh) * P.page_tokens + w0 - page_index(w0) * P.page_tokens;
          unsigned char* kt = smem + C::kTiles + (s * 4 + warp) * 2 * C::kTileBytes;
          unsigned char* sc = smem + C::kScales + (s * 4 + warp) * 2 * C::kScaleBytes;
          uint64_t* bar = &bars[warp][s];
          mbar_expect_tx(bar, 2 * (C::kTileBytes + C::kScaleBytes));
          tma_load_2d(kt, &k_map, bar, 0, row);
          bulk_load(sc, (const unsigned char*)P.k_scale + (size_t)row * (4 * NG), C::kScaleBytes, bar);
          tma_load_2d(kt + C::kTileBytes, &v_map, bar, 0, row);
          bulk_load(sc + C::kScaleBytes, (const unsigned char*)P.v_scale + (size_t)row * (4 * NG), C::kScaleBytes, bar);
        }
      }
      --l_left;
      if (++l_t == lu.T) {
        l_t = 0;
        if (++l_kvh == P.Hkv) {
          l_kvh = 0;
          if (++l_rt == lu.row_tiles) {
            l_rt = 0;
            if (l_left > 0) lu = next_seq(lu);
          }
        }
        ask_pages();
      } else if (l_t == l_page0 + 32) {
        ask_pages();
      }
      if (has) return;
    }
  };
  for (int s = 0; s < C::kStages; ++s) issue_next();

  float o[MT][NT][2];                             // dims (row g, row g + 8 of tile mt) of query row 4 nt + t
  float m_r[NT], l_r[NT], f_r[NT], z[NT][NG];
  int qs[NT][NG];
  float qsf[NT][NG];
  uint32_t qb[D / 32][NT][2];
  // where the lane's row of an ldmatrix stands: (keys 0-7 | 8-15) x (chunk 2c, 2c + 1) of a tile's first 16 keys; 16
  // keys on is 16 rows on, whole periods of the swizzle
  uint32_t at16[RB / 32];
#pragma unroll
  for (int c = 0; c < RB / 32; ++c)
    at16[c] = swizzled<RB>(((lane & 7) + ((lane >> 3) & 1) * 8) * RB + (2 * c + (lane >> 4)) * 16);
  int cs_b = -1;

  for (int done = 0; done < n_steps;) {
    // ---- the unit's query rows: rotated if asked, whole numbers of 16 bits in two bytes
    const int rows = cu.q_len * G, row0 = c_rt * C::kRows, seg = min(cu.T - c_t, n_steps - done);
    const bool turn = P.fused && P.inv_freq != nullptr, fresh = has_new(cu, c_t, seg);
    if (turn && cs_b != cu.b) {
      __syncthreads();
      if (threadIdx.x < D / 2) rotation(cu.base, freq, &cs_s[threadIdx.x], &cs_s[D / 2 + threadIdx.x]);
      cs_b = cu.b;
    }
    __syncthreads();
    auto rotate = [&](float (&a)[D / 32]) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const float cv = cs_s[i * 32 + lane], sv = cs_s[D / 2 + i * 32 + lane];
        const float lo = rotate_lo(a[i], a[i + D / 64], cv, sv);
        a[i + D / 64] = rotate_hi(a[i], a[i + D / 64], cv, sv);
        a[i] = lo;
      }
    };
    if (fresh && warp < 2) {
      // the new token's row: rotated, quantised, into the cache and, for the tile that it belongs to, shared memory
      if (turn && warp == 0) rotate(ta);
      float* row_s = reinterpret_cast<float*>(smem + C::kJoin) + warp * D;      // (no join is under way)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) row_s[32 * i + lane] = ta[i];
      __syncwarp();
      const bool held = t_page >= 0 && t_page < P.n_pages;
      absent_page |= !held;
      const size_t prow = ((size_t)(held ? t_page : 0) * P.Hkv + c_kvh) * P.page_tokens + cu.base - page_index(cu.base) * P.page_tokens;
      uint8_t* dst = (warp == 0 ? P.k_pool : P.v_pool) + prow * RB;
      uint32_t* scale_dst = reinterpret_cast<uint32_t*>(warp == 0 ? P.k_scale : P.v_scale) + prow * NG;
      uint8_t* tile = reinterpret_cast<uint8_t*>(new_codes[warp]);
      quantize_row<BITS>(
          row_s, D, lane,
          [&](int d, uint32_t c) {
            if (BITS == 8) {
              *reinterpret_cast<uint16_t*>(tile + d) = (uint16_t)c;
              if (held) *reinterpret_cast<uint16_t*>(dst + d) = (uint16_t)c;
            } else {
              tile[d / 2] = (uint8_t)c;
              if (held) dst[d / 2] = (uint8_t)c;
            }
          },
          [&](int gr, float s, __nv_bfloat162 sm) {
            const uint32_t w = BITS == 8 ? __float_as_uint(s) : *reinterpret_cast<const uint32_t*>(&sm);
            new_scale[warp][gr] = w;
            if (held) scale_dst[gr] = w;
          });
    }
    signed char* q_s = reinterpret_cast<signed char*>(smem + C::kQ);     // column 2r: high bytes of row r, 2r + 1: low bytes
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = 4 * j + warp;
      float (&a)[D / 32] = qa[j];
      if (turn) rotate(a);
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) amax = max_nan(amax, fabsf(a[i]));
#pragma unroll
      for (int sh = 16; sh > 0; sh >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, sh));
      const bool fine = isfinite(amax) && amax > 1e-30f;       // else zeros; NaN through the factor where not finite
      const float up = fine ? kFixedQ / amax : 0.f;
      int sum[NG];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) sum[gr] = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int v = fine ? __float2int_rn(a[i] * up) : 0;
        sum[BITS == 8 ? 0 : 32 * i / kQuantGroup] += v;
        const int hi = (v + 128) >> 8;             // v = 256 hi + lo, lo in -128 .. 127
        // 4 bits: a word holds eight dims, the even ones in its low halves, the odd ones in its high halves
        const int d = 32 * i + lane, at = BITS == 8 ? d : (d & ~7) + ((d & 1) << 2) + ((d & 7) >> 1);
        q_s[(2 * r) * C::kQStride + at] = (signed char)hi;
        q_s[(2 * r + 1) * C::kQStride + at] = (signed char)(v - (hi << 8));
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        sum[gr] = __reduce_add_sync(0xffffffffu, sum[gr]);
        if (lane == 0) qsum_s[r][gr] = sum[gr];
      }
      if (lane == 0) f_s[r] = fine ? P.sl2 * (amax / kFixedQ) : amax - amax;
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const signed char* qc = q_s + (8 * nt + g) * C::kQStride;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        if (BITS == 8) {                           // dims 32c + 4t .. + 3 and 16 more
          qb[c][nt][0] = *reinterpret_cast<const uint32_t*>(qc + 32 * c + 4 * q4);
          qb[c][nt][1] = *reinterpret_cast<const uint32_t*>(qc + 32 * c + 16 + 4 * q4);
        } else {                                   // dims 32c + 8t + (0, 2, 4, 6 | 1, 3, 5, 7)
          const uint2 w = *reinterpret_cast<const uint2*>(qc + 32 * c + 8 * q4);
          qb[c][nt][0] = w.x;
          qb[c][nt][1] = w.y;
        }
      }
      f_r[nt] = f_s[4 * nt + q4];
      m_r[nt] = -INFINITY;
      l_r[nt] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        qs[nt][gr] = qsum_s[4 * nt + q4][gr];           // (4 bits only)
        qsf[nt][gr] = (float)qs[nt][gr];
        z[nt][gr] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt][nt][0] = o[mt][nt][1] = 0.f;
    }
    const int first_limit = cu.base + row0 / G;    // the last key the unit's first row sees

    for (int st = 0; st < seg; ++st) {
      const int w0 = (c_t + st) * C::kBlockKeys + warp * WK;
      if (w0 >= cu.len) break;
      if (!ring.take(arrived)) break;              // the result is reported as lost; the joins still take place
      const int stage = ring.stage();
      unsigned char* kt = smem + C::kTiles + (stage * 4 + warp) * 2 * C::kTileBytes;
      unsigned char* vt = kt + C::kTileBytes;
      unsigned char* sc = smem + C::kScales + (stage * 4 + warp) * 2 * C::kScaleBytes;

      if (fresh && cu.base >= w0 && cu.base < w0 + WK) {
        // over the row that was loaded
        const int at = cu.base - w0;
        if (lane < RB / 4) {
          const uint32_t off = swizzled<RB>((uint32_t)(at * RB + lane * 4));
          *reinterpret_cast<uint32_t*>(kt + off) = new_codes[0][lane];
          *reinterpret_cast<uint32_t*>(vt + off) = new_codes[1][lane];
        }
        if (lane < NG) {
          reinterpret_cast<uint32_t*>(sc)[at * NG + lane] = new_scale[0][lane];
          reinterpret_cast<uint32_t*>(sc + C::kScaleBytes)[at * NG + lane] = new_scale[1][lane];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // before the next load into this stage
        __syncwarp();
      }

      // ---- scores: keys on the rows (g, g + 8 of each 16), query row 4 nt + t on a lane's column pair
      const uint32_t k_addr = smem_u32(kt), v_addr = smem_u32(vt);
      auto load_scales = [](uint32_t (&w)[NG], const unsigned char* from, int key) {
        if (NG == 2) {
          const uint2 v = reinterpret_cast<const uint2*>(from)[key];
          w[0] = v.x;
          w[NG - 1] = v.y;
        } else {
          w[0] = reinterpret_cast<const uint32_t*>(from)[key];
        }
      };
      float x[KT][NT][2];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        // the two keys' scales
        uint32_t ksc[2][NG];
#pragma unroll
        for (int h = 0; h < 2; ++h) load_scales(ksc[h], sc, 16 * k + 8 * h + g);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          int acc[NT][4];
          if (BITS == 8) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t w[4];
              ldmatrix_x4(w, k_addr + at16[c] + k * 16 * RB);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (c == 0) mma_bytes<true, true, true>(acc[nt], w[0], w[1], w[2], w[3], qb[c][nt][0], qb[c][nt][1]);
                else mma_bytes<true, true, false>(acc[nt], w[0], w[1], w[2], w[3], qb[c][nt][0], qb[c][nt][1]);
              }
            }
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] = acc[nt][2] = 0;
              acc[nt][1] = acc[nt][3] = -8 * qs[nt][gr];
            }
            uint32_t w[4];                         // 64 dims: chunks 2 gr and 2 gr + 1
            ldmatrix_x4(w, k_addr + at16[gr] + k * 16 * RB);
            constexpr uint32_t LO = 0x0f0f0f0fu;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_bytes<false, true, false>(acc[nt], w[2 * h] & LO, w[2 * h + 1] & LO, (w[2 * h] >> 4) & LO,
                                              (w[2 * h + 1] >> 4) & LO, qb[2 * gr + h][nt][0], qb[2 * gr + h][nt][1]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (BITS == 8) {
              const float s = __uint_as_float(ksc[h][0]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) x[k][nt][h] = (float)(acc[nt][2 * h] * 256 + acc[nt][2 * h + 1]) * s;
            } else {
              const float s = __uint_as_float(ksc[h][gr] << 16), mid = __uint_as_float(ksc[h][gr] & 0xffff0000u);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                x[k][nt][h] = fmaf((float)(acc[nt][2 * h] * 256 + acc[nt][2 * h + 1]), s,
                                   gr ? fmaf(mid, qsf[nt][gr], x[k][nt][h]) : mid * qsf[nt][gr]);
              }
            }
          }
        }
      }

      // ---- probabilities against the row's reference m, their sum, and p sv as whole numbers of 16 bits against
      // the step's largest, two bytes in a column pair: the second product's operand (keys on k: 2t, 2t + 8,
      // 2t + 1, 2t + 9 of each 16)
      uint32_t pb[KT][NT][NG];
      float beta[NT][NG];                                   // what the step's integer sums are worth
      auto softmax = [&](auto masked_c) {
        constexpr bool MASKED = decltype(masked_c)::value;
        const unsigned char* scv = sc + C::kScaleBytes;
        float sv[KT][2][NG], low[KT][2][NG];
        bool seen[KT][NT][2];                               // which of the lane's (key, query row) pairs count
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (MASKED) {
            const int limit = min(cu.base + min((row0 + 4 * nt + q4) / G, cu.q_len - 1), cu.len - 1);
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) seen[k][nt][h] = w0 + 16 * k + 8 * h + g <= limit;
          }
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[NG];
            load_scales(w, scv, 16 * k + 8 * h + g);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              if (BITS == 8) {
                sv[k][h][gr] = __uint_as_float(w[gr]);
              } else {
                sv[k][h][gr] = __uint_as_float(w[gr] << 16);
                low[k][h][gr] = fmaf(-8.f, sv[k][h][gr], __uint_as_float(w[gr] & 0xffff0000u));
              }
            }
          }
        float p[KT][NT][2], top[NT][NG];                    // probabilities; the step's largest p sv
        auto exponentials = [&]() {
          bool far = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) top[nt][gr] = 1e-30f;      // below it a step adds nothing that counts
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                p[k][nt][h] = fast_exp2(fmaf(x[k][nt][h], f_r[nt], -m_r[nt]));
                // a key that the row does not see adds nothing (not 0 x NaN)
                if (MASKED && !seen[k][nt][h]) { p[k][nt][h] = 0.f; continue; }
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) top[nt][gr] = max_nan(top[nt][gr], p[k][nt][h] * sv[k][h][gr]);
                far |= p[k][nt][h] > 1e30f;                 // a value's scale may hide how far the score is
              }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
#pragma unroll
              for (int sh = 4; sh <= 16; sh <<= 1) top[nt][gr] = max_nan(top[nt][gr], __shfl_xor_sync(0xffffffffu, top[nt][gr], sh));
              far |= top[nt][gr] > 1048576.f;
            }
          }
          return far;
        };
        if (__any_sync(0xffffffffu, exponentials())) {      // the unit's first step, and hardly ever after
          // the reference moves to the largest s + log2 sv seen so far; a row of zeros (or of values below 127 x
          // 2^-40) must not move it without end, or leave a sum of p that no float32 holds
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float m = m_r[nt];
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (!MASKED || seen[k][nt][h])
#pragma unroll
                  for (int gr = 0; gr < NG; ++gr)
                    m = fmaxf(m, fmaf(x[k][nt][h], f_r[nt], __log2f(fmaxf(sv[k][h][gr], 9.1e-13f))));
#pragma unroll
            for (int sh = 4; sh <= 16; sh <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, sh));
            // (the sum of p may be as far above 1 as the factor is below what a float32 holds: it takes its root twice)
            const float root = m == m_r[nt] ? 1.f : fast_exp2(0.5f * (m_r[nt] - m)), alpha = root * root;
            m_r[nt] = m;
            l_r[nt] = l_r[nt] * root * root;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) z[nt][gr] *= alpha;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) { o[mt][nt][0] *= alpha; o[mt][nt][1] *= alpha; }
          }
          exponentials();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float up[NG];
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            beta[nt][gr] = top[nt][gr] * (1.f / kFixedP);
            up[gr] = __fdividef(kFixedP, top[nt][gr]);
          }
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            l_r[nt] += p[k][nt][0] + p[k][nt][1];
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              uint32_t y[2];                                // low 16 bits: rint(p sv up), by adding 2^23
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                y[h] = __float_as_uint(fmaf(p[k][nt][h] * sv[k][h][gr], up[gr], 8388608.f));
                if (MASKED && !seen[k][nt][h]) y[h] = 0;
                if (BITS == 4) {
                  const float t = fmaf(p[k][nt][h], low[k][h][gr], z[nt][gr]);
                  z[nt][gr] = !MASKED || seen[k][nt][h] ? t : z[nt][gr];
                }
              }
              pb[k][nt][gr] = transpose_8x8(__byte_perm(y[0], y[1], 0x4051));     // (high g, high g + 8 | low g, low g + 8)
            }
          }
        }
      };
      // some row does not see some key of the tile
      if (w0 + WK - 1 > min(first_limit, cu.len - 1)) softmax(std::true_type{});
      else softmax(std::false_type{});
      // ---- O^T += V^T P^T: value dims on the rows, four keys a register
      // 8 bits: rows g and g + 8 of tile mt hold dims 16 mt + 2g and one more; 4 bits: of tile 2c + i dims
      // 32c + 4g + 2i and one more
#pragma unroll
      for (int c = 0; c < RB / 32; ++c) {
        uint32_t even[KT][2], odd[KT][2];                   // bytes 2g and 2g + 1 of chunks 2c, 2c + 1
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          uint32_t w[4];
          ldmatrix_x4_trans(w, v_addr + at16[c] + k * 16 * RB);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            even[k][i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x6240);
            odd[k][i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7351);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int part = 0; part < 8 / BITS; ++part) {
            const int mt = BITS == 8 ? 2 * c + i : 2 * (2 * c + i) + part, gr = BITS == 8 ? 0 : mt * 16 / kQuantGroup;
            int acc[NT][4];
#pragma unroll
            for (int k = 0; k < KT; k += 2) {
              constexpr uint32_t LO = 0x0f0f0f0fu, HI = 0xf0f0f0f0u;
              uint32_t a[4];
              if (BITS == 8) {
                a[0] = even[k][i]; a[1] = odd[k][i]; a[2] = even[k + 1][i]; a[3] = odd[k + 1][i];
              } else {                                      // (the high halves as they stand: 16 times the code)
                const uint32_t u = part ? odd[k][i] : even[k][i], v = part ? odd[k + 1][i] : even[k + 1][i];
                a[0] = u & LO; a[1] = u & HI; a[2] = v & LO; a[3] = v & HI;
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (k == 0) mma_bytes<BITS == 8, false, true>(acc[nt], a[0], a[1], a[2], a[3], pb[k][nt][gr], pb[k + 1][nt][gr]);
                else mma_bytes<BITS == 8, false, false>(acc[nt], a[0], a[1], a[2], a[3], pb[k][nt][gr], pb[k + 1][nt][gr]);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              o[mt][nt][0] = fmaf((float)(acc[nt][0] * 256 + acc[nt][1]), beta[nt][gr], o[mt][nt][0]);
              o[mt][nt][1] = fmaf((float)(acc[nt][2] * 256 + acc[nt][3]), BITS == 8 ? beta[nt][gr] : beta[nt][gr] * 0.0625f,
                                  o[mt][nt][1]);
            }
          }
      }
      ring.release();
      __syncwarp();                                          // every lane has read the stage
      issue_next();
    }

    // ---- the unit's end in this block: the next unit's rows asked for; then lanes, then warps
    const QuantSeq u = cu;                          // (the join below still speaks of this unit)
    const int u_begin = unit_begin, u_kvh = c_kvh;
    done += seg;
    c_t += seg;
    if (c_t == cu.T && done < n_steps) {
      unit_begin += cu.T;
      c_t = 0;
      if (++c_kvh == P.Hkv) {
        c_kvh = 0;
        if (++c_rt == cu.row_tiles) {
          c_rt = 0;
          cu = next_seq(cu);
        }
      }
      fetch(cu, c_rt, c_kvh, 0, n_steps - done);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int sh = 4; sh <= 16; sh <<= 1) {
        l_r[nt] += __shfl_xor_sync(0xffffffffu, l_r[nt], sh);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) z[nt][gr] += __shfl_xor_sync(0xffffffffu, z[nt][gr], sh);
      }
      if (BITS == 4) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o[mt][nt][0] += z[nt][mt * 16 / kQuantGroup];
          o[mt][nt][1] += z[nt][mt * 16 / kQuantGroup];
        }
      }
    }
    float* join = reinterpret_cast<float*>(smem + C::kJoin);
    auto put = [&](int buf) {
      float2* j = reinterpret_cast<float2*>(join + buf * C::kRegs * 32) + lane;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) j[(mt * NT + nt) * 32] = make_float2(o[mt][nt][0], o[mt][nt][1]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        ml_s[buf][nt * 2][lane] = m_r[nt];
        ml_s[buf][nt * 2 + 1][lane] = l_r[nt];
      }
    };
    // (m, l, o) of two parts of a row's keys as one
    auto factors = [](float& m, float& l, float m2, float l2, float& fa, float& fb) {
      const float mx = fmaxf(m, m2);
      const float ra = m == mx ? 1.f : fast_exp2(0.5f * (m - mx)), rb = m2 == mx ? 1.f : fast_exp2(0.5f * (m2 - mx));
      fa = ra * ra;
      fb = rb * rb;
      m = mx;
      l = l * ra * ra + l2 * rb * rb;
    };
    auto add = [&](int buf) {
      const float2* j = reinterpret_cast<const float2*>(join + buf * C::kRegs * 32) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float fa, fb;
        factors(m_r[nt], l_r[nt], ml_s[buf][nt * 2][lane], ml_s[buf][nt * 2 + 1][lane], fa, fb);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float2 v = j[(mt * NT + nt) * 32];
          o[mt][nt][0] = o[mt][nt][0] * fa + v.x * fb;
          o[mt][nt][1] = o[mt][nt][1] * fa + v.y * fb;
        }
      }
    };
    auto join_warps = [&]() {                       // warp 0 ends with the block's sums
      if (warp & 1) put(warp >> 1);
      __syncthreads();
      if (!(warp & 1)) add(warp >> 1);
      if (warp == 2) put(1);
      __syncthreads();
      if (warp == 0) add(1);
    };
    join_warps();
    const int u_end = u_begin + u.T;
    const bool whole = u_begin >= begin && u_end <= end;
    auto store_all = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float inv = 1.f / l_r[nt];
        const int row = row0 + 4 * nt + q4;
        __nv_bfloat16* dst = P.out + (size_t)(u.t0 + row / G) * P.Hq * D + (size_t)(u_kvh * G + row % G) * D + (BITS == 8 ? 2 : 4) * g;
        if (row < rows)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            *reinterpret_cast<uint32_t*>(dst + (BITS == 8 ? 16 * mt : 32 * (mt >> 1) + 2 * (mt & 1))) =
                pack_bf16(o[mt][nt][0] * inv, o[mt][nt][1] * inv);
      }
    };
    if (warp == 0) {
      if (whole) {
        store_all();
      } else {
        float4* seg_out = reinterpret_cast<float4*>(P.scratch + ((size_t)blockIdx.x * 2 + (begin >= u_begin ? 0 : 1)) * C::kSegFloats);
        float r[C::kRegs];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            r[(mt * NT + nt) * 2] = o[mt][nt][0];
            r[(mt * NT + nt) * 2 + 1] = o[mt][nt][1];
          }
#pragma unroll
        for (int i = 0; i < C::kRegs / 4; ++i) __stcg(seg_out + i * 32 + lane, make_float4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          __stcg(reinterpret_cast<float2*>(seg_out + C::kRegs / 4 * 32) + nt * 32 + lane, make_float2(m_r[nt], l_r[nt]));
      }
    }
    if (!whole) {
      // blocks whose share meets this unit: first .. last; the one that comes last joins them in order
      const int first = by_unit ? blockIdx.x - part : block_of(u_begin);
      const int last = by_unit ? first + parts_of(u) - 1 : block_of(u_end - 1);
      // counters are indexed by the unit's first block: a block begins at most one cut unit, whose other
      // segments are the first ones of later blocks
      if (warp == 0) {
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          const int before = atomicAdd(P.counters + first, 1);
          last_s = before == last - first;
          if (before == last - first) P.counters[first] = 0;
        }
      }
      __syncthreads();
      if (last_s) {
        __threadfence();
        // warp w joins segments w, w + 4, ... in order, then the four warps join as above; kAhead segments are
        // asked for together.  (Of the unit's blocks all but the first begin inside the unit.)
        const int first_seg = first * 2 + (by_unit || begin_of(first) >= u_begin ? 0 : 1);
        const float4* segs = reinterpret_cast<const float4*>(P.scratch) + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          m_r[nt] = -INFINITY;
          l_r[nt] = 0.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[mt][nt][0] = o[mt][nt][1] = 0.f;
        }
        constexpr int kAhead = C::kRegs <= 16 ? 4 : 1;
        for (int i0 = first + warp; i0 <= last; i0 += 4 * kAhead) {
          float4 a[kAhead][C::kRegs / 4];
          float2 ml[kAhead][NT];
#pragma unroll
          for (int v = 0; v < kAhead; ++v) {
            const int i = min(i0 + 4 * v, last);
            const float4* s = segs + (size_t)(i == first ? first_seg : 2 * i) * (C::kSegFloats / 4);
#pragma unroll
            for (int r = 0; r < C::kRegs / 4; ++r) a[v][r] = __ldcg(s + r * 32);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              ml[v][nt] = __ldcg(reinterpret_cast<const float2*>(s - lane + C::kRegs / 4 * 32) + nt * 32 + lane);
          }
#pragma unroll
          for (int v = 0; v < kAhead; ++v) {
            if (i0 + 4 * v > last) break;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float fa, fb;
              factors(m_r[nt], l_r[nt], ml[v][nt].x, ml[v][nt].y, fa, fb);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                const int r = (mt * NT + nt) * 2;
                const float4 w = a[v][r / 4];
                o[mt][nt][0] = o[mt][nt][0] * fa + (r & 2 ? w.z : w.x) * fb;
                o[mt][nt][1] = o[mt][nt][1] * fa + (r & 2 ? w.w : w.y) * fb;
              }
            }
          }
        }
        join_warps();
        if (warp == 0) store_all();
      }
    }
  }
  ring.drain(arrived);                            // (empty unless a wait ran out)
  if (absent_page || past_table) atomicOr(P.status, kStatusBadPage);
  if (lane == 0 && ring.expired) atomicOr(P.status, kStatusWaitExpired);
}

// ------------------------------------------------------------------ host
static bool code_map(CUtensorMap* map, const void* pool, long long rows, int row_bytes, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)row_bytes, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUtensorMapSwizzle sw = row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                : row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BITS, int D, int NT>
static int launch_quant(const QuantAttnParams& p, int blocks, cudaStream_t stream) {
  using C = QuantAttn<BITS, D, NT>;
  const long long rows = (long long)p.n_pages * p.Hkv * p.page_tokens;
  CUtensorMap k_map, v_map;
  if (!code_map(&k_map, p.k_pool, rows, C::kRowBytes, C::kWarpKeys) || !code_map(&v_map, p.v_pool, rows, C::kRowBytes, C::kWarpKeys))
    return (int)cudaErrorInvalidValue;
  auto kern = attn_quant_kernel<BITS, D, NT>;
  constexpr int smem = C::kSmem + 1024;
  static bool attr[64] = {};                       // a property of the device's copy of the kernel
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  if (!attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr[dev] = true;
  }
  return (int)launch_kernel(kern, dim3(blocks), dim3(128), smem, stream, p, k_map, v_map);
}

// Column tiles (of four query rows) of a unit for up to `rows` (new tokens x heads of a group) a sequence.
static int column_tiles_of(int rows) { return rows <= 4 ? 1 : rows <= 8 ? 2 : 4; }

template <int BITS, int D>
static int blocks_per_sm(int nt) {
  return nt == 1 ? QuantAttn<BITS, D, 1>::kBlocksPerSM : nt == 2 ? QuantAttn<BITS, D, 2>::kBlocksPerSM : QuantAttn<BITS, D, 4>::kBlocksPerSM;
}

}  // namespace siar

using namespace siar;

SIAR_DEFINE_PDL_SWITCH()

// Blocks of a launch: a block step is the least share.
static int blocks_of(int bits, int B, int Hkv, int D, int rows, int max_kv_len, int sm_count) {
  const int nt = column_tiles_of(rows);
  const int keys = D == 128 && (bits == 8 || nt == 4) ? 128 : 256;
  const long long steps = (long long)B * Hkv * ((rows + 4 * nt - 1) / (4 * nt)) * ((max_kv_len + keys - 1) / keys);
  const long long most = (long long)sm_count * (bits == 8 ? D == 128 ? blocks_per_sm<8, 128>(nt) : blocks_per_sm<8, 64>(nt)
                                                          : D == 128 ? blocks_per_sm<4, 128>(nt) : blocks_per_sm<4, 64>(nt));
  return (int)(steps < most ? (steps > 0 ? steps : 1) : most);
}

// What every launch on a GPU of so many SMs finds room in: counters (int32), and floats of scratch behind them.
extern "C" long long siar_attn_quant_counters(int sm_count) { return 3ll * sm_count; }
extern "C" long long siar_attn_quant_scratch_floats(int sm_count) {
  constexpr long long narrow = 3 * QuantAttn<8, 64, 1>::kSegFloats, wide = 2 * QuantAttn<8, 128, 4>::kSegFloats;
  static_assert(QuantAttn<8, 64, 1>::kBlocksPerSM == 3 && QuantAttn<8, 128, 4>::kBlocksPerSM == 2, "the most of either");
  return 2ll * sm_count * (narrow > wide ? narrow : wide);
}

// What tells one capture of a stream from another (0: the stream is not being captured).
extern "C" unsigned long long siar_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id) != cudaSuccess) return 0;
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// Attention of the batch's new tokens over the quantised cache.  fused: one new token a sequence, whose
// query and key are rotated here (inv_freq; nullptr: not rotated) and whose key and value are stored
// (write_kv) and attended to; else the tokens' rows are in the cache and the queries are as they are to be
// used, in qkv or (q16 not nullptr; qkv is not read then) as siar_rope_quantize_q16 leaves them.  Sequences with more than
// most_new new tokens are passed over (max_q_len and max_kv_len are those of the others).  counters:
// siar_attn_quant_counters int32 zeros, left zero; scratch: siar_attn_quant_scratch_floats floats.
static int siar_attn_quant_of(int bits, const void* qkv, const void* q16, const float* q_factor, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                               const int* block_table, const int* slot_ids, const int* q_start, const int* base_len,
                               const float* inv_freq, void* out, int* counters, float* scratch, int B, int Hq, int Hkv, int D,
                               int page_tokens, int max_pages, int n_pages, int max_q_len, int max_kv_len, int sm_count,
                               int fused, int write_kv, int most_new, float scale, int* status, void* stream) {
  if (B == 0 || max_q_len == 0) return 0;
  if (Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128) || page_tokens <= 0 || page_tokens % 64 != 0 || (bits != 8 && bits != 4) ||
      n_pages <= 0 || max_pages <= 0 || max_kv_len <= 0 || sm_count <= 0 || (fused && (max_q_len != 1 || q16 != nullptr)) ||
      (long long)n_pages * Hkv * page_tokens >= (1ll << 31) || (long long)max_pages * page_tokens >= (1ll << 31))
    return (int)cudaErrorInvalidValue;
  QuantAttnParams p = {(const __nv_bfloat16*)qkv, (const __half*)q16, q_factor, (uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids,
                       q_start, base_len, inv_freq, (__nv_bfloat16*)out, scratch, counters, status, B, Hq, Hkv, page_tokens,
                       max_pages, n_pages, (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1, fused,
                       write_kv, most_new, scale * 1.4426950408889634f};
  cudaStream_t s = (cudaStream_t)stream;
  const int blocks = blocks_of(bits, B, Hkv, D, max_q_len * (Hq / Hkv), max_kv_len, sm_count);
  const int nt = column_tiles_of(max_q_len * (Hq / Hkv));
#define SIAR_GO(BITS, DIM)                                                                     \
  return nt == 1 ? launch_quant<BITS, DIM, 1>(p, blocks, s) : nt == 2 ? launch_quant<BITS, DIM, 2>(p, blocks, s) \
                                                                      : launch_quant<BITS, DIM, 4>(p, blocks, s)
  if (bits == 8) {
    if (D == 64) { SIAR_GO(8, 64); }
    SIAR_GO(8, 128);
  }
  if (D == 64) { SIAR_GO(4, 64); }
  SIAR_GO(4, 128);
#undef SIAR_GO
}
SIAR_TAKES_WORDS(siar_attn_quant)
