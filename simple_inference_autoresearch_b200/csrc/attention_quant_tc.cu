// Attention of many new tokens a sequence (prompts, chunks of prompts) over a cache held in 8 or 4 bits, on the
// 5th-generation tensor cores, in three kernels behind the one that stores the new tokens:
//
//   widen_tiles     the batch's keys and values as float16 tiles of 64 positions, each tile times a power of two that
//                   brings what its scales allow to 2^9 .. 2^10: a value keeps 11 bits (a bfloat16 cache has 8), and
//                   the factor costs nothing, because a key tile's goes into the factor of its scores and a value tile's
//                   into the exponent;
//   attn_quant_tc   the kernel of attention_tc.cu (its roles, rings and tensor-memory layout are described there)
//                   on float16 operands: queries as float16 with a power of two of their own, P in float16 against a
//                   reference that leaves it 32 binary orders of range.  A block has 128 rows of one kv head's queries,
//                   so that two blocks share an SM: one's softmax runs under the other's products.  (Blocks of 256 rows,
//                   one an SM: a prompt of 2,048 tokens 74 us, of 128 rows 67.)  Where the rows are too few to fill
//                   the GPU the keys of a block of rows are cut into parts;
//   attn_quant_join adds the parts up.
//
// Roundings to fewer bits: queries, keys, values and P to float16 (11 bits of each; the sum of P takes the unrounded ones).
// They are small beside the result's own to bfloat16: relative error against 64 bits 0.00177 for the chunk below, 0.00169
// with 32 bits throughout.
//
// All of it, with the kernel that stores the tokens, takes 64 us for a prompt of 2,048 tokens (4 bits, 32 heads on 8, 128
// dims; its products at the measured matrix rate 21 us) and 99 us for a chunk of 515 on 8,191 held (8 bits, 24 on 8; 32
// us).  The chunk's kernels one by one: 9 us storing, 16 widening, 75 the products, 10 joining (they overlap at their
// ends).  In the products' kernel neither the tensor pipe (37 %) nor the exponentials (37 %) are busy all the time: a
// tile is a chain scores -> largest -> exponentials -> P -> O, some 1,700 cycles for a block alone and 1,900 with two on an
// SM, at 1.7 GHz.  (With scores and P.V issued by one thread of a warp, and a load a tile for its factors, the two took
// 66 and 104 us.)  Products are fed from shared memory at 128 bytes a clock and read Q again for every 64 keys, 512
// clocks a tile.  Tried and no faster: two threads a row (131 us), all key tiles shared out evenly over two blocks an
// SM (104 to 111, the prompt 68 to 73), four-stage rings.  Reading the cache back as bfloat16 pages for the bfloat16
// kernel took 87 and 199 us, with 2.5 times the rounding error.
#include "kv_quant.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

namespace siar {

constexpr int kRows = 128;       // query rows per block
constexpr int kKeys = 64;        // keys per tile
constexpr int kStages = 2;       // K and V rings
constexpr int smem_bytes(int hd) { return kRows * hd * 2 + kStages * 2 * kKeys * hd * 2; }
constexpr uint32_t kTmemCols = 256;                 // S[buf]: 64 columns each from 0; O: head_dim from kOColumn
constexpr uint32_t kOColumn = 128;
constexpr float kHeadroom = 8.f, kRescaleGap = 7.f; // log2 of where p of the largest score starts, and of what it may grow by
constexpr int kBlocksPerSM = 2;
constexpr int kThreads = 256;                       // TMA warp, scores, a spare, P.V, four softmax warps

// What the softmax has to know of a key tile and its value tile.
struct TileInfo {
  float k_factor;                // a key is the tile's float16 times this power of two
  float v_log2;                  // a value is the tile's float16 times 2^v_log2
  unsigned long long bad[2];     // bit r: the value of position r is not a number (in its first, second run of 64 dims)
};

// The sequences of a launch, by their places in the batch.
constexpr int kMostSeqs = 64;
struct SeqList {
  unsigned short b[kMostSeqs];
};

struct QuantTcParams {
  __nv_bfloat16* out;
  float* scratch;                // parts of rows: [tokens x heads][splits][head_dim + 8]
  const TileInfo* tiles;         // [tiles][Hkv]
  const int* seq_tiles;          // [listed sequences]: the sequence's first tile, and how many it has
  const float* q_factor;         // [tokens][Hq]
  const int* q_start;
  const int* base_len;
  int* status;
  int Hq, Hkv, splits;
  float sl2;                     // scale * log2(e)
};

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Two float32 operations in one instruction.
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves_of(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 32 bytes, a whole sector, in one store (a thread owns a row: narrower stores leave sectors half written).
__device__ __forceinline__ void store_sector(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Instruction descriptor of kind::f16 with float16 operands: D float32, A K-major, M = 128, N = n; B K-major or MN-major.
__host__ __device__ constexpr uint32_t instr_desc_f16(int n, bool b_mn_major = false) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Key tiles of the block of rows that begins at row0: up to the last key its last row sees, and what the sequence has.
__host__ __device__ inline int key_tiles(int base, int q_len, int row0, int G, int tile_rows, int held) {
  const int last = min(q_len * G, row0 + tile_rows) - 1;
  return min((base + last / G + 1 + kKeys - 1) / kKeys, held);
}
template <int kHd>
__global__ void __launch_bounds__(kThreads, kBlocksPerSM)
attn_quant_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const QuantTcParams prm, const __grid_constant__ SeqList seqs) {
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t q_full;
  __shared__ __align__(8) uint64_t s_full[2], p_full[2], pv_full[2];
  // keys and values have rings of their own: a key stage is free again as soon as the scores that
  // read it are done, a value stage only after P.V, a step later, so each is asked for as early as it can be
  __shared__ __align__(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  constexpr int kHalves = kHd / 64;                  // 64-dim (128-byte) column blocks of a row
  constexpr int kQBytes = kRows * kHd * 2;           // 16 KiB per half
  constexpr int kTileBytes = kKeys * kHd * 2;        // 8 KiB per half
  pdl_wait();
  asm volatile("fence.proxy.async.global;" ::: "memory");      // queries and tiles that the kernels in front stored, for the TMA
  // blocks with the most keys (the last rows, of all sequences and heads) start first: the tail of the grid is made
  // of short blocks
  const int part = blockIdx.x % prm.splits, kvh = blockIdx.x / prm.splits % prm.Hkv, at = blockIdx.x / prm.splits / prm.Hkv;
  const int b = seqs.b[at];
  const int G = prm.Hq / prm.Hkv;
  const int tile_rows = (kRows / G) * G;             // rows in use: whole tokens only
  const int t0 = prm.q_start[b];
  const int q_len = prm.q_start[b + 1] - t0;
  const int rows_total = q_len * G;
  const int row0 = (gridDim.y - 1 - blockIdx.y) * tile_rows;
  if (row0 >= rows_total) return;
  const int base = prm.base_len[b];
  const int all_tiles = key_tiles(base, q_len, row0, G, tile_rows, prm.seq_tiles[2 * at + 1]);
  const int parts = min(prm.splits, all_tiles);
  if (part >= parts) return;
  const int tile0 = all_tiles * part / parts, nt_max = all_tiles * (part + 1) / parts - tile0;
  const int seq_first = prm.seq_tiles[2 * at];        // the sequence's first tile of the widened cache

  const uint32_t dyn = smem_u32(smem_dyn);
  unsigned char* sm = smem_dyn + ((1024u - (dyn & 1023u)) & 1023u);
  unsigned char* q_s = sm;                                   // [half][128 rows][64 dims]
  unsigned char* k_s = q_s + kQBytes;                        // [stage][half][64 keys][64 dims]
  unsigned char* v_s = k_s + kStages * kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);                      // the softmax warps (no barrier among them: one that gave up would hold the rest)
      mbar_init(&pv_full[i], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_base_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Tensor memory is taken behind the wait (all kernels in front have given theirs back) and in front of this, so the next
  // kernel starts only when every block here has its columns: a product takes its own in front of its wait, and holding them
  // beside a block that still asks for columns it would wait for that block without end.
  pdl_launch_dependents();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
  const bool dead = (*(volatile int*)prm.status & kStatusWaitExpired) != 0;

#define SIAR_FAIL()                                   \
  {                                                   \
    abort_flag = 1;                                   \
    atomicOr(prm.status, kStatusWaitExpired);         \
  }
#define SIAR_ABORTED() (*(volatile int*)&abort_flag != 0)

  if (dead) {
    // another block already reported an expired wait: do nothing
  } else if (warp == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tmQ) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV) : "memory");
      mbar_expect_tx(&q_full, tile_rows * kHd * 2);      // a box is tile_rows packed rows (the rest of the tile stays as it was: masked rows)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        tma_load_3d(q_s + h * (kQBytes / kHalves), &tmQ, &q_full, 64 * h, kvh * G, t0 + row0 / G);
      int issued_k = 0, issued_v = 0;
      for (int i = 0; i < nt_max; ++i) {
        const int s = i % kStages;
        const uint32_t ph = ((i / kStages) & 1) ^ 1;
        const int row = ((seq_first + tile0 + i) * prm.Hkv + kvh) * kKeys;
        if (!mbar_wait(&k_empty[s], ph) || SIAR_ABORTED()) { SIAR_FAIL(); break; }
        mbar_expect_tx(&k_full[s], kTileBytes);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          tma_load_2d(k_s + s * kTileBytes + h * (kTileBytes / kHalves), &tmK, &k_full[s], 64 * h, row);
        issued_k = i + 1;
        if (!mbar_wait(&v_empty[s], ph) || SIAR_ABORTED()) { SIAR_FAIL(); break; }
        mbar_expect_tx(&v_full[s], kTileBytes);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          tma_load_2d(v_s + s * kTileBytes + h * (kTileBytes / kHalves), &tmV, &v_full[s], 64 * h, row);
        issued_v = i + 1;
      }
      // Copies in flight land before the block leaves, whoever gives up and when: the last ones may be under way when every
      // load has been issued.
      mbar_wait(&q_full, 0);
      for (int i = max(0, issued_k - kStages); i < issued_k; ++i) mbar_wait(&k_full[i % kStages], (i / kStages) & 1);
      for (int i = max(0, issued_v - kStages); i < issued_v; ++i) mbar_wait(&v_full[i % kStages], (i / kStages) & 1);
    }
  } else if (warp == 1 || warp == 3) {
    // ---------------- MMA issue: warp 1 the scores, warp 3 P.V.  One thread issues; the whole warp walks along, so that all it
    // computes is the same in every lane and stays in uniform registers, where the products take their operands
    // from (issue under lane == 0: 75 cycles a product more).
    auto wait = [](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
    const bool chosen = elect_one();
    // descriptors differ in their low word only (the address field, in units of 16 bytes)
    const uint32_t hi_k = (uint32_t)(smem_desc_sw128(0) >> 32);
    const uint32_t hi_v = (uint32_t)(smem_desc_sw128_mn(0, kTileBytes / kHalves) >> 32);
    const uint32_t q_lo = (uint32_t)smem_desc_sw128(smem_u32(q_s));
    const uint32_t k_lo = (uint32_t)smem_desc_sw128(smem_u32(k_s));
    const uint32_t v_lo = (uint32_t)smem_desc_sw128_mn(smem_u32(v_s), kTileBytes / kHalves);
    bool ok = true;
    if (warp == 1) {
      ok = wait(&q_full, 0);
      for (int i = 0; i < nt_max && ok; ++i) {
        // the buffer is free when the P.V that read P from it is done
        ok = wait(&k_full[i % kStages], (i / kStages) & 1) && (i < 2 || wait(&pv_full[i & 1], ((i - 2) >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        if (chosen) {
          // S[i & 1] = Q K_i^T over the 64-dim halves, 4 steps of 16 dims (32 bytes) in each
          constexpr uint32_t idesc = instr_desc_f16(kKeys);
          const uint32_t ks = k_lo + (uint32_t)((i % kStages) * (kTileBytes >> 4));
#pragma unroll
          for (int kk = 0; kk < kHd / kUmmaK; ++kk)
            umma_f16_words(tmem_base + (uint32_t)((i & 1) * kKeys), q_lo + (uint32_t)((kk / 4) * (kQBytes / kHalves >> 4) + (kk % 4) * 2), hi_k,
                           ks + (uint32_t)((kk / 4) * (kTileBytes / kHalves >> 4) + (kk % 4) * 2), hi_k, idesc, kk > 0 ? 1u : 0u);
          umma_commit(&s_full[i & 1]);
          umma_commit(&k_empty[i % kStages]);       // the key stage is free once these scores are done
        }
        __syncwarp();
      }
    } else {
      for (int i = 0; i < nt_max && ok; ++i) {
        ok = wait(&v_full[i % kStages], (i / kStages) & 1) && wait(&p_full[i & 1], (i >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (chosen) {
          // O += P V: 4 steps of 16 keys; V rows (keys) are 128 bytes of one dim half, 8-row groups 1024 bytes apart,
          // the two dim halves 8 KiB apart.  P sits in tensor memory, in the first 32 columns of the scores it was made
          // from.
          constexpr uint32_t idesc = instr_desc_f16(kHd, true);
          const uint32_t vs = v_lo + (uint32_t)((i % kStages) * (kTileBytes >> 4));
#pragma unroll
          for (int t = 0; t < kKeys / kUmmaK; ++t)
            umma_f16_tmem_a(tmem_base + kOColumn, tmem_base + (uint32_t)((i & 1) * kKeys + t * 8), vs + (uint32_t)(t * (2048 >> 4)),
                            hi_v, idesc, (i > 0 || t > 0) ? 1u : 0u);
          umma_commit(&pv_full[i & 1]);
          umma_commit(&v_empty[i % kStages]);
        }
        __syncwarp();
      }
    }
    if (!ok && chosen) SIAR_FAIL();
  } else if (warp >= 4) {
    // ---------------- softmax: one thread per row
    const int quad = warp & 3;                 // the tensor-memory lanes this warp may touch
    const int row = quad * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t tmem_o = tmem_base + kOColumn + lane_base;
    const int rg = row0 + row;
    const bool mine = row < min(tile_rows, rows_total - row0);
    const int kv_end = mine ? base + rg / G + 1 : 0;
    const size_t out_row = (size_t)(t0 + (mine ? rg / G : 0)) * prm.Hq + kvh * G + (mine ? rg % G : 0);
    const float row_scale = prm.sl2 * prm.q_factor[out_row];       // of a raw score, times the tile's key factor
    const TileInfo* info = prm.tiles + ((size_t)seq_first + tile0) * prm.Hkv + kvh;
    float k_factors = 0.f, v_logs = 0.f;        // lane l: of tile l of 32
    unsigned bad_tiles = 0;
    const int n_tiles = nt_max;
    float m_used = -INFINITY, l = 0.f;
    unsigned poisoned = 0;                      // runs of 64 dims in which the row sees a value that is not a number
    bool ok = true;
    for (int i = 0; i < n_tiles; ++i) {
      const int j0 = (tile0 + i) * kKeys;
      if (i % 32 == 0) {
        const TileInfo* t = info + (size_t)min(i + lane, n_tiles - 1) * prm.Hkv;
        k_factors = t->k_factor;
        v_logs = t->v_log2;
        bad_tiles = __ballot_sync(0xffffffffu, (t->bad[0] | t->bad[1]) != 0);
      }
      const float sl2 = row_scale * __shfl_sync(0xffffffffu, k_factors, i % 32);
      const float v_log2 = __shfl_sync(0xffffffffu, v_logs, i % 32);
      if (!mbar_wait(&s_full[i & 1], (i >> 1) & 1) || SIAR_ABORTED()) { ok = false; break; }
      tc_fence_after();
      const uint32_t tmem_s = tmem_base + (uint32_t)((i & 1) * kKeys) + lane_base;
      uint32_t sr[64];
      SIAR_TMEM_LD_32(tmem_s, sr);
      {
        uint32_t* hi = sr + 32;
        SIAR_TMEM_LD_32(tmem_s + 32, hi);
      }
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (j0 + kKeys > kv_end) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (j0 + j >= kv_end) sr[j] = 0xff800000u;      // -inf
      }
      if ((bad_tiles >> (i % 32)) & 1) {
        // values that are not numbers stand as zeros in the tile (0 x NaN would reach rows that do not see them)
        const TileInfo* t = info + (size_t)i * prm.Hkv;
        const int n = kv_end - j0;
        const unsigned long long seen = n >= kKeys ? ~0ull : n > 0 ? (1ull << n) - 1ull : 0ull;
        poisoned |= (t->bad[0] & seen ? 1u : 0u) | (t->bad[1] & seen ? 2u : 0u);
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(sr[j + e]));
      }
      const float raw = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // The reference is kHeadroom below the largest s + log2(value factor) so far, so that p is at most
      // 2^(kHeadroom + kRescaleGap) and float16 holds it down to 2^-32 of the largest.  A row whose raw scores are
      // all hidden (or NaN) has no maximum yet.
      const float m_new = fmaxf(m_used, raw * sl2 + v_log2 - kHeadroom);
      const bool need = m_new > m_used + kRescaleGap;      // also true for the first finite maximum
      if (i > 0 && __any_sync(0xffffffffu, need)) {
        // O may be touched once the previous tile's P.V has completed
        if (!mbar_wait(&pv_full[(i - 1) & 1], ((i - 1) >> 1) & 1) || SIAR_ABORTED()) { ok = false; break; }
        tc_fence_after();
        // (the sum of p may be as far above 1 as the factor is below what a float32 holds: it takes its root twice)
        const float root = need ? (m_used == -INFINITY ? 0.f : ex2(0.5f * (m_used - m_new))) : 1.f, alpha = root * root;
        l = l * root * root;
#pragma unroll 1
        for (int ch = 0; ch < kHd / 32; ++ch) {
          uint32_t o[32];
          SIAR_TMEM_LD_32(tmem_o + ch * 32, o);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          SIAR_TMEM_ST_32(tmem_o + ch * 32, o);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      if (need) m_used = m_new;
      const float neg_m = m_used == -INFINITY ? 0.f : v_log2 - m_used;
      // P = 2^(s c - m) as float16 pairs, written over the first 32 columns of the scores in tensor
      // memory (this thread holds its whole row in registers by now).  The next scores for this
      // buffer are issued after the P.V that reads P is done.
      unsigned long long sum[4] = {0ull, 0ull, 0ull, 0ull};
      const unsigned long long by = pair_of(sl2, sl2), off = pair_of(neg_m, neg_m);
      uint32_t pw[32];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = halves_of(fma_pair(pair_of(__uint_as_float(sr[c * 8 + 2 * e]), __uint_as_float(sr[c * 8 + 2 * e + 1])), by, off));
          const float p0 = ex2(x.x), p1 = ex2(x.y);
          sum[e] = add_pair(sum[e], pair_of(p0, p1));
          pw[c * 4 + e] = pack_f16x2(p0, p1);
        }
      }
      SIAR_TMEM_ST_32(tmem_s, pw);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      const float2 both = halves_of(add_pair(add_pair(sum[0], sum[1]), add_pair(sum[2], sum[3])));
      l += (both.x + both.y) * __int_as_float((127 - (int)v_log2) << 23);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i & 1]);
    }
    if (ok) ok = mbar_wait(&pv_full[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1);
    if (!ok) {
      SIAR_FAIL();
    } else {
      tc_fence_after();
      const float nan = __int_as_float(0x7fc00000);
      const float inv = parts == 1 ? 1.f / l : 1.f;
      __nv_bfloat16* dst = prm.out + out_row * kHd;
      float* partial = prm.scratch + (out_row * prm.splits + part) * (kHd + 8);      // (reference, sum), then the sums of values
#pragma unroll 1
      for (int ch = 0; ch < kHd / 32; ++ch) {
        uint32_t o[32];
        SIAR_TMEM_LD_32(tmem_o + ch * 32, o);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (!mine) continue;
        const float f = (poisoned >> (ch * 32 / 64)) & 1 ? nan : inv;
        if (parts == 1) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 pk;
            pk.x = pack_bf16x2(__uint_as_float(o[j]) * f, __uint_as_float(o[j + 1]) * f);
            pk.y = pack_bf16x2(__uint_as_float(o[j + 2]) * f, __uint_as_float(o[j + 3]) * f);
            pk.z = pack_bf16x2(__uint_as_float(o[j + 4]) * f, __uint_as_float(o[j + 5]) * f);
            pk.w = pack_bf16x2(__uint_as_float(o[j + 6]) * f, __uint_as_float(o[j + 7]) * f);
            *reinterpret_cast<uint4*>(dst + ch * 32 + j) = pk;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[j + e]) * f;
            store_sector(partial + 8 + ch * 32 + j, v);
          }
        }
      }
      if (mine && parts > 1) __stcg(reinterpret_cast<float2*>(partial), make_float2(m_used, l));
    }
  }
#undef SIAR_FAIL
#undef SIAR_ABORTED
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base_slot, kTmemCols);
  }
}


// ------------------------------------------------------------------ widening
// grid (tiles of the longest sequence, Hkv, listed sequences), 256 threads.  Rows behind a sequence's last token are zeros.
template <int D, int BITS>
__global__ void __launch_bounds__(256)
widen_tiles_kernel(const uint8_t* k_pool, const uint8_t* v_pool, const void* k_scale, const void* v_scale,
                   const int* block_table, const int* slot_ids, const int* q_start, const int* base_len, __half* k_out,
                   __half* v_out, TileInfo* tiles, int* seq_tiles, const __grid_constant__ SeqList seqs, int Hkv, int page_tokens,
                   int max_pages, int n_pages, int tiles_out, int* __restrict__ status) {
  constexpr int NG = BITS == 8 ? 1 : D / kQuantGroup;
  pdl_launch_dependents();
  __shared__ float bound_s[4];
  __shared__ unsigned bad_s[2][4];                   // [run][32 rows of K, K, V, V]
  __shared__ int first_s;
  pdl_wait();
  const int tile = blockIdx.x, kvh = blockIdx.y, at = blockIdx.z, b = seqs.b[at];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cap = max_pages * page_tokens;
  auto length_of = [&](int i) { return max(0, min(base_len[i] + q_start[i + 1] - q_start[i], min(cap, (int)gridDim.x * kKeys))); };
  const int total = length_of(b), mine = (total + kKeys - 1) / kKeys;
  const int slot = slot_ids[b];
  // the page is asked for before the tiles in front are counted
  const int pos = tile * kKeys;
  int page = tile < mine ? block_table[(size_t)slot * max_pages + pos / page_tokens] : 0;
  if (warp == 7) {
    int sum = 0;
    for (int i = lane; i < at; i += 32) sum += (length_of(seqs.b[i]) + kKeys - 1) / kKeys;
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) first_s = sum;
  }
  if (tile == 0 && kvh == 0 && threadIdx.x == 0 && base_len[b] + q_start[b + 1] - q_start[b] > total)
    atomicOr(status, total == cap ? kStatusBadPage : kStatusLengthPastGrid);
  const bool absent = page < 0 || page >= n_pages;
  if (absent) {
    page = 0;
    if (threadIdx.x == 0) atomicOr(status, kStatusBadPage);
  }
  const size_t row0 = ((size_t)page * Hkv + kvh) * page_tokens + pos % page_tokens;
  const int held = absent ? 0 : min(kKeys, total - pos);
  // what the scales allow, per tile: warps 0 and 1 the keys, 2 and 3 the values
  if (warp < 4) {
    const int r = (warp & 1) * 32 + lane;
    const uint32_t* sc = reinterpret_cast<const uint32_t*>(warp < 2 ? k_scale : v_scale) + (row0 + r) * NG;
    float most = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t w = tile < mine && r < held ? sc[g] : 0u;
      const float s = __uint_as_float(BITS == 8 ? w : w << 16);
      const float of_run = BITS == 8 ? 127.f * s : 8.f * s + fabsf(__uint_as_float(w & 0xffff0000u));
      const unsigned bad = __ballot_sync(0xffffffffu, !(of_run <= 3.4e38f));
      if (lane == 0) bad_s[g][warp] = bad;
      if (of_run <= 3.4e38f) most = fmaxf(most, of_run);
    }
    most = warp_max(most);
    if (lane == 0) bound_s[warp] = most;
  }
  __syncthreads();
  const int first = first_s;
  if (tile == 0 && kvh == 0 && threadIdx.x == 0) {
    seq_tiles[2 * at] = first;
    seq_tiles[2 * at + 1] = max(0, min(mine, tiles_out - first));
    if (first + mine > tiles_out) atomicOr(status, kStatusLengthPastGrid);      // host lengths that fall short
  }
  if (tile >= mine || first + tile >= tiles_out) return;
  // The power of two that brings the bound to 2^9 .. 2^10.  At most 2^40 (below a bound of 2^-31 a tile's values keep
  // fewer bits), 2^20 for a tile of zeros: the softmax takes p against the largest p x value, so the sum of p of a tile of
  // next to nothing beside one of very large values has to stand within the range of a float32.
  float up[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const float bound = fmaxf(bound_s[2 * kv], bound_s[2 * kv + 1]);
    const int e = (int)(__float_as_uint(bound) >> 23) - 127;
    up[kv] = __uint_as_float((uint32_t)(max(-120, min(bound > 0.f ? 40 : 20, 9 - e)) + 127) << 23);
  }
  const size_t out_row0 = ((size_t)(first + tile) * Hkv + kvh) * kKeys;
  if (threadIdx.x == 0) {
    TileInfo t;
    t.k_factor = 1.f / up[0];
    t.v_log2 = -(float)((int)(__float_as_uint(up[1]) >> 23) - 127);
    t.bad[0] = bad_s[0][2] | (unsigned long long)bad_s[0][3] << 32;
    t.bad[1] = NG == 2 ? bad_s[NG - 1][2] | (unsigned long long)bad_s[NG - 1][3] << 32 : D == 128 ? t.bad[0] : 0ull;
    tiles[(size_t)(first + tile) * Hkv + kvh] = t;
  }
  constexpr int PER_ROW = D / 16;
#pragma unroll 1
  for (int idx = threadIdx.x; idx < 2 * kKeys * PER_ROW; idx += 256) {
    const bool is_k = idx < kKeys * PER_ROW;
    const int i = is_k ? idx : idx - kKeys * PER_ROW;
    const int r = i / PER_ROW, d = (i % PER_ROW) * 16;
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
    if (r < held) {
      const uint8_t* src = (is_k ? k_pool : v_pool) + ((row0 + r) * D + d) * BITS / 8;
      const uint32_t w = reinterpret_cast<const uint32_t*>(is_k ? k_scale : v_scale)[(row0 + r) * NG + (NG == 1 ? 0 : d / kQuantGroup)];
      const float f = up[is_k ? 0 : 1];
      float s = __uint_as_float(BITS == 8 ? w : w << 16) * f, m = BITS == 8 ? 0.f : __uint_as_float(w & 0xffff0000u) * f;
      if (!is_k && !(fabsf(s) <= 3.4e38f && fabsf(m) <= 3.4e38f)) s = m = 0.f;      // reported by `bad`
      if (BITS == 8) {
        const uint4 c = *reinterpret_cast<const uint4*>(src);
        const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = (__uint_as_float(__byte_perm(cw[e >> 2] ^ 0x80808080u, 0x4b000000u, 0x7440 + (e & 3))) - 8388736.f) * s;
      } else {
        const uint2 c = *reinterpret_cast<const uint2*>(src);
        const uint32_t cw[2] = {c.x, c.y};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = fmaf(__uint_as_float(((cw[e >> 3] >> (4 * (e & 7))) & 15u) | 0x4b000000u) - 8388616.f, s, m);
      }
    }
    uint4 o[2];
    uint32_t* ow = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int e = 0; e < 8; ++e) ow[e] = pack_f16x2(x[2 * e], x[2 * e + 1]);
    uint4* dst = reinterpret_cast<uint4*>((is_k ? k_out : v_out) + (out_row0 + r) * D + d);
    dst[0] = o[0];
    dst[1] = o[1];
  }
}

// ------------------------------------------------------------------ parts of rows
// One warp a row (token, head); rows of sequences that are not listed are passed over.
template <int D>
__global__ void __launch_bounds__(256)
attn_quant_join_kernel(const float* scratch, __nv_bfloat16* out, const int* seq_tiles, const int* q_start, const int* base_len,
                       const __grid_constant__ SeqList seqs, int listed, int N, int B, int Hq, int Hkv, int splits) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = row / Hq, head = row % Hq;
  if (t >= N) return;
  const int G = Hq / Hkv, tile_rows = (kRows / G) * G;
  int b = 0;
  for (int hi = B - 1; b < hi;) {
    const int mid = (b + hi + 1) >> 1;
    if (q_start[mid] <= t) b = mid; else hi = mid - 1;
  }
  const int t0 = q_start[b], q_len = q_start[b + 1] - t0;
  if (t < t0 || t >= t0 + q_len) return;
  int at = -1;
#pragma unroll
  for (int i = 0; i < kMostSeqs; i += 32) {
    const unsigned hit = __ballot_sync(0xffffffffu, i + lane < listed && seqs.b[i + lane] == b);
    if (hit != 0) at = i + __ffs(hit) - 1;
  }
  if (at < 0) return;
  const int rg = (t - t0) * G + head % G;
  const int parts = min(splits, key_tiles(base_len[b], q_len, rg / tile_rows * tile_rows, G, tile_rows, seq_tiles[2 * at + 1]));
  if (parts < 2) return;
  const float* part = scratch + (size_t)row * splits * (D + 8);
  float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int p = 0; p < parts; ++p, part += D + 8) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(part));
    const float mx = fmaxf(m, ml.x), ra = m == mx ? 1.f : ex2(0.5f * (m - mx)), rb = ml.x == mx ? 1.f : ex2(0.5f * (ml.x - mx));
    const float fa = ra * ra, fb = rb * rb;
    l = l * ra * ra + ml.y * rb * rb;
    m = mx;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = acc[i] * fa + __ldcg(part + 8 + i * 32 + lane) * fb;
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) out[(size_t)row * D + i * 32 + lane] = __float2bfloat16_rn(acc[i] / l);
}

// ------------------------------------------------------------------ host side
static bool f16_map(const void* ptr, long long rows, int hd, CUtensorMap* out) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t gdim[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  const cuuint64_t gstride[1] = {(cuuint64_t)hd * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)kKeys}, ones[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), gdim, gstride, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The queries as [tokens, Hq heads, head_dim], seen in boxes of floor(128/G) tokens x G heads x 64 dims.
static bool query_map(const void* q, int n_tokens, int Hq, int Hkv, int hd, CUtensorMap* out) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int G = Hq / Hkv;
  const cuuint64_t gdim[3] = {(cuuint64_t)hd, (cuuint64_t)Hq, (cuuint64_t)n_tokens};
  const cuuint64_t gstride[2] = {(cuuint64_t)hd * 2, (cuuint64_t)Hq * hd * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(kRows / G)}, ones[3] = {1, 1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), gdim, gstride, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
static int launch_tc(const CUtensorMap& tmQ, const CUtensorMap& tmK, const CUtensorMap& tmV, const QuantTcParams& prm, dim3 grid,
                     const SeqList& seqs, int listed, int N, int B, cudaStream_t s) {
  constexpr int smem = smem_bytes(D) + 1024;
  static bool attr[64] = {};                       // a property of the device's copy of the kernel
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  if (!attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_quant_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr[dev] = true;
  }
  const cudaError_t e = launch_kernel(attn_quant_tc_kernel<D>, grid, dim3(kThreads), smem, s, tmQ, tmK, tmV, prm, seqs);
  if (e != cudaSuccess || prm.splits == 1) return (int)e;
  return (int)launch_kernel(attn_quant_join_kernel<D>, dim3((unsigned)(((long long)N * prm.Hq + 7) / 8)), dim3(256), 0, s,
                            (const float*)prm.scratch, prm.out, prm.seq_tiles, prm.q_start, prm.base_len, seqs, listed, N, B, prm.Hq, prm.Hkv,
                            prm.splits);
}

static bool seq_list(const int* ids, int n, int B, SeqList* out) {
  if (n <= 0 || n > kMostSeqs) return false;
  for (int i = 0; i < n; ++i) {
    if (ids[i] < 0 || ids[i] >= B || ids[i] > 65535) return false;
    out->b[i] = (unsigned short)ids[i];
  }
  for (int i = n; i < kMostSeqs; ++i) out->b[i] = 0;
  return true;
}

}  // namespace siar

using namespace siar;

SIAR_DEFINE_PDL_SWITCH()

// Into how many parts the keys of a block of 128 rows are cut, for `blocks` of them of up to `longest` (on average
// `average`) key tiles.  Measured on B200 at 128 dims: a block alone on its SM takes 7 us and 0.95 us a tile, two on
// every SM 0.66 us a tile and SM, the last round a third of a block more; parts (`row_floats` floats each) are written and
// read again at 3.6 TB/s by a kernel of its own.  A chunk of 128 tokens on 8,000 held (32 heads on 8): one part 139 us, 8
// parts 54; a chunk of 515 on 8,191 (24 on 8): parts 1, 2, 3, 4, 5, 6, 8 take 134, 101, 114, 99, 97, 109, 109 us (the rule
// takes 4); a prompt of 2,048: one part 64 us, two over 100.  Where its estimate is furthest off: 1,000 tokens of 8 heads on 1 on
// 20,000 held take 127 us with the rule's 7 parts, 103 with 4; 256 on 60,000 343 with 13, 318 with 4.  The constants are those
// of 128 dims; at 64 dims (us, the rule's choice and the best of 1 to 16): 128 on 8,000 44 (10 parts) and 37 (8), 515 on
// 8,191 89 (6) and 80 (5), 300 on 2,000 30 (3) and 30, four times 64 on 16,000 93 (11) and 91 (6), prompts one part and best.
extern "C" int siar_attn_quant_tc_parts(int blocks, int longest, float average, long long row_floats, int sms) {
  int best = 1;
  float best_cost = 1e30f;
  for (int parts = 1; parts <= 16 && parts <= longest; ++parts) {
    const float tiles = (float)((longest + parts - 1) / parts);
    const float alone = 7.f + 0.95f * tiles, shared = (float)blocks * average * 0.66f / (float)sms + 0.35f * (7.f + 1.3f * tiles);
    const float cost = (alone > shared ? alone : shared) + (parts > 1 ? 4.f + (float)parts * (float)row_floats * 8.f / 3.6e6f : 0.f);
    if (cost < best_cost) { best_cost = cost; best = parts; }
  }
  return best;
}

extern "C" int siar_attn_quant_tc_tile_info_bytes(void) { return (int)sizeof(TileInfo); }

extern "C" int siar_attn_quant_tc_most_seqs(void) { return kMostSeqs; }

// The keys and values of `listed` of the batch's B sequences (ids: their places in it, on the host) as float16 tiles of 64
// positions, sequence after sequence: k_out, v_out [tiles_out, Hkv, 64, D], tiles [tiles_out, Hkv]
// (siar_attn_quant_tc_tile_info_bytes each), seq_tiles [listed, 2].
static int siar_widen_tiles_of(int bits, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                                const int* block_table, const int* slot_ids, const int* q_start, const int* base_len, void* k_out,
                                void* v_out, void* tiles, int* seq_tiles, const int* ids, int listed, int B, int Hkv, int D,
                                int page_tokens, int max_pages, int n_pages, int tiles_out, int max_kv_len, int* status, void* stream) {
  if (B == 0) return 0;
  SeqList seqs;
  if (!seq_list(ids, listed, B, &seqs) || (bits != 8 && bits != 4) || (D != 64 && D != 128) || Hkv > 65535 || page_tokens <= 0 || page_tokens % kKeys != 0 ||
      max_kv_len <= 0 || n_pages <= 0 || (long long)max_pages * page_tokens >= (1ll << 31))
    return (int)cudaErrorInvalidValue;
  auto go = [&](auto kernel) {
    return (int)launch_kernel(kernel, dim3((max_kv_len + kKeys - 1) / kKeys, Hkv, listed), dim3(256), 0, (cudaStream_t)stream,
                              (const uint8_t*)k_pool, (const uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids, q_start, base_len,
                              (__half*)k_out, (__half*)v_out, (TileInfo*)tiles, seq_tiles, seqs, Hkv, page_tokens, max_pages, n_pages,
                              tiles_out, status);
  };
  if (bits == 8) return D == 64 ? go(widen_tiles_kernel<64, 8>) : go(widen_tiles_kernel<128, 8>);
  return D == 64 ? go(widen_tiles_kernel<64, 4>) : go(widen_tiles_kernel<128, 4>);
}
SIAR_TAKES_WORDS(siar_widen_tiles)

// q [N, Hq, D] float16 with q_factor [N, Hq]; out [N, Hq * D] bfloat16; scratch: with splits > 1 N * Hq * splits * (D + 8)
// floats.  splits: parts into which the keys of a block of rows are cut.  ids, listed, and what follows from
// them in seq_tiles, as siar_widen_tiles had them; max_q_len is that of the listed sequences, rows of others stay as they are.
static int siar_attn_quant_tc_of(const void* q, const float* q_factor, const void* k_tiles, const void* v_tiles, const void* tiles,
                                  const int* seq_tiles, const int* q_start, const int* base_len, void* out, float* scratch, const int* ids,
                                  int listed, int N, int B, int Hq, int Hkv, int D, int tiles_out, int max_q_len, int splits, float scale, int* status,
                                  void* stream) {
  if (B == 0 || max_q_len == 0 || N == 0) return 0;
  SeqList seqs;
  if (!seq_list(ids, listed, B, &seqs) || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128) || Hq / Hkv > kRows || splits < 1 || !(scale > 0.f) ||
      (long long)tiles_out * Hkv * kKeys >= (1ll << 31))
    return (int)cudaErrorInvalidValue;
  CUtensorMap tmQ, tmK, tmV;
  const long long rows = (long long)tiles_out * Hkv * kKeys;
  if (!query_map(q, N, Hq, Hkv, D, &tmQ) || !f16_map(k_tiles, rows, D, &tmK) || !f16_map(v_tiles, rows, D, &tmV))
    return (int)cudaErrorInvalidValue;
  const QuantTcParams prm = {(__nv_bfloat16*)out, scratch, (const TileInfo*)tiles, seq_tiles, q_factor, q_start, base_len, status, Hq,
                             Hkv, splits, scale * 1.4426950408889634f};
  const int G = Hq / Hkv, block_rows = (kRows / G) * G;
  const long long across = (long long)splits * Hkv * listed, down = (max_q_len * (long long)G + block_rows - 1) / block_rows;
  if (across >= (1ll << 31) || down > 65535) return (int)cudaErrorInvalidValue;
  const dim3 grid((unsigned)across, (unsigned)down);
  return D == 64 ? launch_tc<64>(tmQ, tmK, tmV, prm, grid, seqs, listed, N, B, (cudaStream_t)stream)
                 : launch_tc<128>(tmQ, tmK, tmV, prm, grid, seqs, listed, N, B, (cudaStream_t)stream);
}
SIAR_TAKES_WORDS(siar_attn_quant_tc)
