// bfloat16 attention of a few new tokens a sequence over a cache held in 8 or 4 bits (formats: top of
// kv_quant.cu): single tokens of a decode step, with their rotary encoding and cache write inside, and
// short runs of tokens already stored.  head_dim 64 or 128, any group size, pages of a multiple of 64.
//
// Mathematics.  The codes go through the tensor cores as the small whole numbers they are; scales
// enter outside the products:
//   8 bits  s_j = sk_j (q . ck_j),                            out = sum_j (p_j sv_j) cv_j / sum_j p_j
//   4 bits  s_j = sum_g sk_jg (q_g . (ck_jg - 8)) + mk_jg sum(q_g),
//           out_g = (sum_j (p_j sv_jg) (cv_jg - 8) + sum_j p_j mv_jg) / sum_j p_j
// with one pass over the keys and a running reference of the exponent.  A code becomes a float16 by
// placing its bits in the mantissa of 1024 (0x6400 | u = 1024 + u); for keys the constant this adds is
// taken off in the accumulator's start value, for values (whose sums run over thousands of keys) from
// the operand, exactly.  q is scaled by a power of two per row and rounded once to float16 (11 bits where
// bfloat16 keeps 8); p_j sv_j is at most 2^8 by choice of the reference (the running maximum of
// s_j + log2 sv_j, moved only when a product would pass 2^8) and rounded once to float16.  Scores,
// statistics and sums are 32 bits.
//
// Shape.  The products are taken transposed, keys (then value dims) on the MMA's 16 rows and the query
// heads that share a kv head on its 8 columns: half the instructions of heads on the rows, and P moves
// from one product to the other by movmatrix.  What bounds it is memory: a key and value of a head are
// 264 bytes (8 bits, head_dim 128) or 144 (4 bits).
//
// Work is cut evenly: all (sequence, kv head) units' key tiles stand in one row that is shared out over two
// blocks an SM, so unequal lengths leave no tail; a warp's loads (TMA, its own ring of stages, the scales
// along with the codes) run on across the border between two units.  A unit that was cut is joined in
// block order by the block that finishes it last.
#include "attention_mma.cuh"
#include "kv_quant.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace siar {

struct QuantAttnParams {
  const __nv_bfloat16* qkv;      // [N, (Hq + 2 Hkv) D]
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
  float sl2;                     // scale * log2(e)
};

template <int BITS, int D, int NT>
struct QuantAttn {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kWarpKeys = D == 128 ? 32 : 64;                // keys per warp and step
  static constexpr int kBlockKeys = 4 * kWarpKeys;
  static constexpr int kTileBytes = kWarpKeys * kRowBytes;
  static constexpr int kGroups = BITS == 8 ? 1 : D / kQuantGroup;
  static constexpr int kScaleBytes = kWarpKeys * 4 * kGroups;        // float32, or (scale, mid) bfloat16 per run
  // what two blocks an SM leave room for
  static constexpr int kStages = kTileBytes < 4096 ? (NT == 1 ? 5 : 4) : (NT == 1 ? 3 : 2);
  static constexpr int kRows = 8 * NT;                               // query rows of a unit
  static constexpr int kMT = D / 16;                                 // row tiles of the value product
  static constexpr int kQStride = D + 8;                             // float16 elements per query row in shared memory
  static constexpr int kRegs = kMT * NT * 4;                         // accumulators of a lane
  // shared memory
  static constexpr int kTiles = 0;                                   // [stages][warp][K | V]
  static constexpr int kScales = kTiles + kStages * 4 * 2 * kTileBytes;
  static constexpr int kJoin = kScales + kStages * 4 * 2 * kScaleBytes;   // [2][kRegs][32] floats
  static constexpr int kQ = kJoin + 2 * kRegs * 32 * 4;
  static constexpr int kSmem = kQ + kRows * kQStride * 2;
  static constexpr int kSegFloats = (kRegs + 4 * NT) * 32;           // accumulators, maxima, sums
};

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<uint32_t*>(&r);
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

// One sequence's units: (row tile, kv head), all of T block steps.
struct QuantSeq {
  int b, base, t0, q_len, slot, len, T, row_tiles;
};

template <int BITS, int D, int NT>
__global__ void __launch_bounds__(128, 2)
attn_quant_kernel(const __grid_constant__ QuantAttnParams P, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map) {
  using C = QuantAttn<BITS, D, NT>;
  constexpr int WK = C::kWarpKeys, KT = WK / 16, RB = C::kRowBytes, NG = C::kGroups, MT = C::kMT;
  pdl_launch_dependents();
  extern __shared__ unsigned char smem_base[];
  unsigned char* smem = smem_base + ((1024 - (smem_u32(smem_base) & 1023)) & 1023);     // the swizzle pattern's period
  __shared__ __align__(8) uint64_t bars[4][C::kStages];
  __shared__ float cs_s[D];                       // cosines, sines of the new token's position
  __shared__ float row_s[D];                      // the new token's key, then value
  __shared__ float f_s[C::kRows], qsum_s[C::kRows][NG];
  __shared__ float ml_s[2][NT * 4][32];
  __shared__ int last_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q4 = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
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
    s.T = (s.len + C::kBlockKeys - 1) / C::kBlockKeys;
    s.row_tiles = (s.q_len * G + C::kRows - 1) / C::kRows;
    return s;
  };
  // ---- this block's share [begin, end) of all block steps, and the sequence it begins in
  auto steps_of = [&](int b) {
    const QuantSeq s = load_seq(b);
    return (long long)s.T * s.row_tiles * P.Hkv;
  };
  long long total = 0;
  for (int b = lane; b < P.B; b += 32) total += steps_of(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  // at least one step a block: a block without one would be waited for by the join of a unit around it
  const int nb = (int)min((long long)gridDim.x, total);
  if ((int)blockIdx.x >= nb) return;
  const long long begin = total * blockIdx.x / nb, end = total * (blockIdx.x + 1) / nb;
  QuantSeq cu;                                    // unit that is computed: sequence, row tile, kv head, step
  int c_rt, c_kvh, c_t;
  long long unit_begin;                           // first step of the current unit in the whole row
  {
    long long before = 0;
    int b0 = 0;
    while (true) {                                // 32 sequences at a time
      long long mine = b0 + lane < P.B ? steps_of(b0 + lane) : 0, incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + incl > begin);
      if (past != 0 || b0 + 32 >= P.B) {
        const int at = past != 0 ? __ffs(past) - 1 : 31;
        before += __shfl_sync(0xffffffffu, incl - mine, at);
        cu = load_seq(min(b0 + at, P.B - 1));
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      b0 += 32;
    }
    const int in_seq = (int)(begin - before), unit = in_seq / cu.T;
    c_t = in_seq % cu.T;
    c_rt = unit / P.Hkv;
    c_kvh = unit % P.Hkv;
    unit_begin = begin - c_t;
  }
  const int n_steps = (int)(end - begin);

  // ---- this warp's loads: the same walk, ahead of the computation
  QuantSeq lu = cu;
  int l_rt = c_rt, l_kvh = c_kvh, l_t = c_t, l_left = n_steps;
  int issued = 0, consumed = 0;
  bool absent_page = false;
  auto page_index = [&](int pos) { return P.page_shift >= 0 ? pos >> P.page_shift : pos / P.page_tokens; };
  auto next_seq = [&](const QuantSeq& s) {        // the next sequence that has steps (there is one)
    int b = s.b + 1;
    QuantSeq n = load_seq(b);
    while (n.T * n.row_tiles == 0) n = load_seq(++b);
    return n;
  };
  auto page_of = [&]() {                          // page of the load cursor's tile; asked for a step before its use
    const int w0 = l_t * C::kBlockKeys + warp * WK;
    return l_left > 0 && w0 < lu.len ? P.block_table[(size_t)lu.slot * P.max_pages + page_index(w0)] : 0;
  };
  int page_ahead = page_of();
  auto issue_next = [&]() {
    while (l_left > 0) {
      const int w0 = l_t * C::kBlockKeys + warp * WK;
      const bool has = w0 < lu.len;
      if (has) {
        int page = page_ahead;
        if (page < 0 || page >= P.n_pages) { absent_page = true; page = 0; }
        if (lane == 0) {
          const int s = issued % C::kStages;
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
        ++issued;
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
      }
      page_ahead = page_of();
      if (has) return;
    }
  };
  for (int s = 0; s < C::kStages; ++s) issue_next();

  float o[MT][NT][4];
  float m_r[NT][2], l_r[NT][2], f_r[NT][2], z[NT][2][NG], qs[NT][2][NG];
  uint32_t qb[D / 16][NT][2];
  bool expired = false;
  const size_t qkv_row = (size_t)(P.Hq + 2 * P.Hkv) * D;
  int cs_b = -1;

  for (int done = 0; done < n_steps;) {
    // ---- the unit's query rows: rotated if asked, scaled by a power of two, float16
    const int rows = cu.q_len * G, row0 = c_rt * C::kRows;
    if (P.fused && cs_b != cu.b && P.inv_freq != nullptr) {
      __syncthreads();
      if (threadIdx.x < D / 2) rotation(cu.base, P.inv_freq[threadIdx.x], &cs_s[threadIdx.x], &cs_s[D / 2 + threadIdx.x]);
      cs_b = cu.b;
    }
    __syncthreads();
    __half* q_s = reinterpret_cast<__half*>(smem + C::kQ);
    for (int r = warp; r < C::kRows; r += 4) {
      const int row = row0 + r;
      float a[D / 64], c[D / 64], amax = 0.f;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        a[i] = c[i] = 0.f;
        if (row < rows) {
          const __nv_bfloat16* src = P.qkv + (size_t)(cu.t0 + row / G) * qkv_row + (size_t)(c_kvh * G + row % G) * D + i * 32 + lane;
          a[i] = __bfloat162float(src[0]);
          c[i] = __bfloat162float(src[D / 2]);
          if (P.fused && P.inv_freq != nullptr) {
            const float cv = cs_s[i * 32 + lane], sv = cs_s[D / 2 + i * 32 + lane];
            const float lo = rotate_lo(a[i], c[i], cv, sv);
            c[i] = rotate_hi(a[i], c[i], cv, sv);
            a[i] = lo;
          }
        }
        amax = fmaxf(amax, fmaxf(fabsf(a[i]), fabsf(c[i])));
      }
      amax = warp_max(amax);
      // the row's largest element goes to [2^10, 2^11): what float16 then loses at the small end is
      // 2^-35 of it
      int ex = 0;
      if (amax > 0.f && isfinite(amax)) frexpf(amax, &ex);
      const float up = ldexpf(1.f, max(-100, min(100, 11 - ex)));
      float sum[2] = {0.f, 0.f};                   // of the rounded elements, by halves of the head
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const __half ha = __float2half_rn(a[i] * up), hc = __float2half_rn(c[i] * up);
        q_s[r * C::kQStride + i * 32 + lane] = ha;
        q_s[r * C::kQStride + D / 2 + i * 32 + lane] = hc;
        sum[0] += __half2float(ha);
        sum[1] += __half2float(hc);
      }
      sum[0] = warp_sum(sum[0]);
      sum[1] = warp_sum(sum[1]);
      if (lane == 0) {
        f_s[r] = P.sl2 / up;
        if (NG == 2) { qsum_s[r][0] = sum[0]; qsum_s[r][NG - 1] = sum[1]; }
        else qsum_s[r][0] = sum[0] + sum[1];
      }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const __half* qr = q_s + (8 * nt + g) * C::kQStride;
      if (BITS == 8) {
        // k slots (2t, 2t+1 | 2t+8, 2t+9) of chunk c hold dims 16c + 4t + (0, 1 | 2, 3)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const uint2 w = *reinterpret_cast<const uint2*>(qr + 16 * c + 4 * q4);
          qb[c][nt][0] = w.x;
          qb[c][nt][1] = w.y;
        }
      } else {
        // steps 2c and 2c + 1 hold, of a word's eight dims 32c + 8t + i, (0, 4 | 1, 5) and (2, 6 | 3, 7);
        // their codes stand four bits up in the mantissa, hence the sixteenth
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const __half* w = qr + 32 * c + 8 * q4;
          const __half2 k16 = __float2half2_rn(0.0625f);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const __half2 v = __hmul2(__halves2half2(w[h], w[h + 4]), k16);
            qb[2 * c + (h >> 1)][nt][h & 1] = *reinterpret_cast<const uint32_t*>(&v);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * q4 + e;
        f_r[nt][e] = f_s[r];
        m_r[nt][e] = -INFINITY;
        l_r[nt][e] = 0.f;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          qs[nt][e][gr] = qsum_s[r][gr];
          z[nt][e][gr] = 0.f;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
    const int first_limit = cu.base + row0 / G;    // the last key the unit's first row sees

    const int seg = min(cu.T - c_t, n_steps - done);
    for (int st = 0; st < seg; ++st) {
      const int w0 = (c_t + st) * C::kBlockKeys + warp * WK;
      if (w0 >= cu.len) break;
      const int stage = consumed % C::kStages;
      if (!expired && !mbar_wait(&bars[warp][stage], (consumed / C::kStages) & 1)) expired = true;
      unsigned char* kt = smem + C::kTiles + (stage * 4 + warp) * 2 * C::kTileBytes;
      unsigned char* vt = kt + C::kTileBytes;
      unsigned char* sc = smem + C::kScales + (stage * 4 + warp) * 2 * C::kScaleBytes;

      if (P.fused && P.write_kv && cu.base >= w0 && cu.base < w0 + WK && cu.base < cap) {
        // the new token's row: rotated, quantised, into the cache and over the row that was loaded
        const int at = cu.base - w0;
        const int page = P.block_table[(size_t)cu.slot * P.max_pages + cu.base / P.page_tokens];
        const bool held = page >= 0 && page < P.n_pages;
        absent_page |= !held;
        const size_t prow = ((size_t)(held ? page : 0) * P.Hkv + c_kvh) * P.page_tokens + cu.base % P.page_tokens;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          const __nv_bfloat16* src = P.qkv + (size_t)cu.t0 * qkv_row + (size_t)(P.Hq + kv * P.Hkv + c_kvh) * D;
          for (int i = lane; i < D / 2; i += 32) {
            const float a = __bfloat162float(src[i]), c = __bfloat162float(src[i + D / 2]);
            const bool turn = kv == 0 && P.inv_freq != nullptr;
            row_s[i] = turn ? rotate_lo(a, c, cs_s[i], cs_s[D / 2 + i]) : a;
            row_s[i + D / 2] = turn ? rotate_hi(a, c, cs_s[i], cs_s[D / 2 + i]) : c;
          }
          __syncwarp();
          uint8_t* dst = (kv == 0 ? P.k_pool : P.v_pool) + prow * RB;
          float* s8 = reinterpret_cast<float*>(kv == 0 ? P.k_scale : P.v_scale) + prow;
          __nv_bfloat162* s4 = reinterpret_cast<__nv_bfloat162*>(kv == 0 ? P.k_scale : P.v_scale) + prow * NG;
          unsigned char* tile = kv == 0 ? kt : vt;
          unsigned char* scl = sc + kv * C::kScaleBytes + at * 4 * NG;
          quantize_row<BITS>(
              row_s, D, lane,
              [&](int d, uint32_t c) {
                const uint32_t off = swizzled<RB>((uint32_t)(at * RB + d * BITS / 8));
                if (BITS == 8) {
                  *reinterpret_cast<uint16_t*>(tile + off) = (uint16_t)c;
                  if (held) *reinterpret_cast<uint16_t*>(dst + d) = (uint16_t)c;
                } else {
                  tile[off] = (uint8_t)c;
                  if (held) dst[d / 2] = (uint8_t)c;
                }
              },
              [&](int gr, float s, __nv_bfloat162 sm) {
                if (BITS == 8) {
                  *reinterpret_cast<float*>(scl) = s;
                  if (held) *s8 = s;
                } else {
                  reinterpret_cast<__nv_bfloat162*>(scl)[gr] = sm;
                  if (held) s4[gr] = sm;
                }
              });
          __syncwarp();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // before the next load into this stage
      }

      // ---- scores: keys on the rows (g, g + 8 of each 16), query rows 2t, 2t + 1 on the columns
      const uint32_t k_addr = smem_u32(kt), v_addr = smem_u32(vt);
      const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8, lch = lane >> 4;     // ldmatrix: (keys 0-7 | 8-15) x (chunk, next)
      float x[KT][NT][4];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const float* sk8 = reinterpret_cast<const float*>(sc) + 16 * k + g;
        const uint32_t* sk4 = reinterpret_cast<const uint32_t*>(sc) + (16 * k + g) * NG;
        if (BITS == 8) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[nt][0] = acc[nt][2] = -1152.f * qs[nt][0][0];
            acc[nt][1] = acc[nt][3] = -1152.f * qs[nt][1][0];
          }
#pragma unroll
          for (int c = 0; c < D / 16; c += 2) {
            uint32_t w[4];
            ldmatrix_x4(w, k_addr + swizzled<RB>((16 * k + lrow) * RB + (c + lch) * 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a0 = __byte_perm(w[2 * h], 0x64646464u, 0x4140), a2 = __byte_perm(w[2 * h], 0x64646464u, 0x4342);
              const uint32_t a1 = __byte_perm(w[2 * h + 1], 0x64646464u, 0x4140), a3 = __byte_perm(w[2 * h + 1], 0x64646464u, 0x4342);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16_16816(acc[nt], a0, a1, a2, a3, qb[c + h][nt][0], qb[c + h][nt][1]);
            }
          }
          const float s_lo = sk8[0], s_hi = sk8[8];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            x[k][nt][0] = acc[nt][0] * s_lo;
            x[k][nt][1] = acc[nt][1] * s_lo;
            x[k][nt][2] = acc[nt][2] * s_hi;
            x[k][nt][3] = acc[nt][3] * s_hi;
          }
        } else {
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] = acc[nt][2] = -72.f * qs[nt][0][gr];
              acc[nt][1] = acc[nt][3] = -72.f * qs[nt][1][gr];
            }
            uint32_t w[4];
            ldmatrix_x4(w, k_addr + swizzled<RB>((16 * k + lrow) * RB + (2 * gr + lch) * 16));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t lo = w[2 * h], hi = w[2 * h + 1];
              constexpr uint32_t M = 0x00f000f0u, E = 0x64006400u;
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const uint32_t a0 = ((s ? lo >> 4 : lo << 4) & M) | E, a1 = ((s ? hi >> 4 : hi << 4) & M) | E;
                const uint32_t a2 = ((s ? lo >> 8 : lo) & M) | E, a3 = ((s ? hi >> 8 : hi) & M) | E;
                const int st2 = 2 * (2 * gr + h) + s;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_16816(acc[nt], a0, a1, a2, a3, qb[st2][nt][0], qb[st2][nt][1]);
              }
            }
            const uint32_t sm_lo = sk4[gr], sm_hi = sk4[8 * NG + gr];
            const float s_lo = __uint_as_float(sm_lo << 16), mid_lo = __uint_as_float(sm_lo & 0xffff0000u);
            const float s_hi = __uint_as_float(sm_hi << 16), mid_hi = __uint_as_float(sm_hi & 0xffff0000u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float q0 = qs[nt][0][gr], q1 = qs[nt][1][gr];
              const float b0 = gr ? x[k][nt][0] : 0.f, b1 = gr ? x[k][nt][1] : 0.f;
              const float b2 = gr ? x[k][nt][2] : 0.f, b3 = gr ? x[k][nt][3] : 0.f;
              x[k][nt][0] = fmaf(acc[nt][0], s_lo, fmaf(mid_lo, q0, b0));
              x[k][nt][1] = fmaf(acc[nt][1], s_lo, fmaf(mid_lo, q1, b1));
              x[k][nt][2] = fmaf(acc[nt][2], s_hi, fmaf(mid_hi, q0, b2));
              x[k][nt][3] = fmaf(acc[nt][3], s_hi, fmaf(mid_hi, q1, b3));
            }
          }
        }
      }

      // ---- probabilities: value scales of this lane's keys (g, g + 8 of each 16), exponentials, sums, and P as
      // the second product's operand (keys on k, query rows on n)
      uint32_t pb[KT][NT][NG][2];
      auto softmax = [&](auto masked_c) {
        constexpr bool MASKED = decltype(masked_c)::value;
        const unsigned char* scv = sc + C::kScaleBytes;
        float sv[KT][2][NG], mv[KT][2][NG], top[KT][2];
        bool seen[KT][NT][4];                               // which of the lane's (key, query row) pairs count
        if (MASKED) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int limit = min(cu.base + min((row0 + 8 * nt + 2 * q4 + e) / G, cu.q_len - 1), cu.len - 1);
#pragma unroll
              for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) seen[k][nt][2 * h + e] = w0 + 16 * k + 8 * h + g <= limit;
            }
        }
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = 16 * k + 8 * h + g;
            const bool in = !MASKED || w0 + key < cu.len;
            if (BITS == 8) {
              sv[k][h][0] = in ? reinterpret_cast<const float*>(scv)[key] : 0.f;
              top[k][h] = sv[k][h][0];
            } else {
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) {
                const uint32_t sm = in ? reinterpret_cast<const uint32_t*>(scv)[key * NG + gr] : 0u;
                sv[k][h][gr] = __uint_as_float(sm << 16);
                mv[k][h][gr] = __uint_as_float(sm & 0xffff0000u);
                top[k][h] = gr ? fmaxf(top[k][h], sv[k][h][gr]) : sv[k][h][gr];
              }
            }
            // a row of zeros (or of values below 127 x 2^-100) must not lift the reference without end
            top[k][h] = fmaxf(top[k][h], 7.9e-31f);
          }
        float p[KT][NT][4];
        auto exponentials = [&]() {                         // returns the largest p sv
          float most = 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float v = fast_exp2(fmaf(x[k][nt][e], f_r[nt][e & 1], -m_r[nt][e & 1]));
                if (MASKED && !seen[k][nt][e]) v = 0.f;
                p[k][nt][e] = v;
                most = fmaxf(most, v * top[k][e >> 1]);
              }
          return most;
        };
        if (__any_sync(0xffffffffu, exponentials() > 256.f)) {
          // move the reference to the largest s + log2 sv seen so far (the first tile, and rarely after)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = m_r[nt][e];
#pragma unroll
              for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if (!MASKED || seen[k][nt][2 * h + e])
                    mx = fmaxf(mx, fmaf(x[k][nt][2 * h + e], f_r[nt][e], __log2f(top[k][h])));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float alpha = mx == m_r[nt][e] ? 1.f : fast_exp2(m_r[nt][e] - mx);
              m_r[nt][e] = mx;
              l_r[nt][e] *= alpha;
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) z[nt][e][gr] *= alpha;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) { o[mt][nt][e] *= alpha; o[mt][nt][e + 2] *= alpha; }
            }
          exponentials();
        }
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            l_r[nt][0] += p[k][nt][0] + p[k][nt][2];
            l_r[nt][1] += p[k][nt][1] + p[k][nt][3];
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                // a key that the row does not see adds nothing, not 0 x NaN
                v[e] = !MASKED || seen[k][nt][e] ? p[k][nt][e] * sv[k][e >> 1][gr] : 0.f;
                if (BITS == 4)
                  z[nt][e & 1][gr] = !MASKED || seen[k][nt][e] ? fmaf(p[k][nt][e], mv[k][e >> 1][gr], z[nt][e & 1][gr])
                                                               : z[nt][e & 1][gr];
              }
              pb[k][nt][gr][0] = transpose_8x8(pack_f16(v[0], v[1]));
              pb[k][nt][gr][1] = transpose_8x8(pack_f16(v[2], v[3]));
            }
          }
      };
      // some row does not see some key of the tile
      if (w0 + WK - 1 > min(first_limit, cu.len - 1)) softmax(std::true_type{});
      else softmax(std::false_type{});
      // ---- O^T += V^T P^T: value dims on the rows
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (BITS == 8) {
          // rows g and g + 8 of tile c hold dims 16c + 2g and 16c + 2g + 1
#pragma unroll
          for (int c = 0; c < D / 16; c += 2) {
            uint32_t w[4];
            ldmatrix_x4_trans(w, v_addr + swizzled<RB>((16 * k + lrow) * RB + (c + lch) * 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              constexpr uint32_t K1152 = 0x64806480u;        // 1024 + 128
              const uint32_t a0 = h2_sub(__byte_perm(w[2 * h], 0x64646464u, 0x4240), K1152);
              const uint32_t a1 = h2_sub(__byte_perm(w[2 * h], 0x64646464u, 0x4341), K1152);
              const uint32_t a2 = h2_sub(__byte_perm(w[2 * h + 1], 0x64646464u, 0x4240), K1152);
              const uint32_t a3 = h2_sub(__byte_perm(w[2 * h + 1], 0x64646464u, 0x4341), K1152);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[c + h][nt], a0, a1, a2, a3, pb[k][nt][0][0], pb[k][nt][0][1]);
            }
          }
        } else {
          // rows g and g + 8 of tile 2c + h hold dims 32c + 4g + 2h and one more
#pragma unroll
          for (int c = 0; c < D / 32; c += 2) {
            uint32_t w[4];
            ldmatrix_x4_trans(w, v_addr + swizzled<RB>((16 * k + lrow) * RB + (c + lch) * 16));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              constexpr uint32_t LO = 0x000f000fu, HI = 0x00f000f0u, E = 0x64006400u;
              constexpr uint32_t K1032 = 0x64086408u, K16TH = 0x2c002c00u, KM72 = 0xd480d480u;   // 1032, 1/16, -72
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t u = h ? w[2 * i] >> 8 : w[2 * i], v = h ? w[2 * i + 1] >> 8 : w[2 * i + 1];
                const uint32_t a0 = h2_sub((u & LO) | E, K1032), a1 = h2_fma((u & HI) | E, K16TH, KM72);
                const uint32_t a2 = h2_sub((v & LO) | E, K1032), a3 = h2_fma((v & HI) | E, K16TH, KM72);
                const int mt = 2 * (c + i) + h, gr = mt * 16 / kQuantGroup;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_16816(o[mt][nt], a0, a1, a2, a3, pb[k][nt][gr][0], pb[k][nt][gr][1]);
              }
            }
          }
        }
      }
      ++consumed;
      __syncwarp();                                          // every lane has read the stage
      issue_next();
    }

    // ---- the unit's end in this block: lanes, then warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int sh = 4; sh <= 16; sh <<= 1) {
          l_r[nt][e] += __shfl_xor_sync(0xffffffffu, l_r[nt][e], sh);
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) z[nt][e][gr] += __shfl_xor_sync(0xffffffffu, z[nt][e][gr], sh);
        }
        if (BITS == 4) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            o[mt][nt][e] += z[nt][e][mt * 16 / kQuantGroup];
            o[mt][nt][e + 2] += z[nt][e][mt * 16 / kQuantGroup];
          }
        }
      }
    float* join = reinterpret_cast<float*>(smem + C::kJoin);
    auto put = [&](int buf) {
      float* j = join + buf * C::kRegs * 32 + lane;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) j[((mt * NT + nt) * 4 + e) * 32] = o[mt][nt][e];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          ml_s[buf][nt * 4 + e][lane] = m_r[nt][e];
          ml_s[buf][nt * 4 + 2 + e][lane] = l_r[nt][e];
        }
    };
    auto add = [&](int buf) {
      const float* j = join + buf * C::kRegs * 32 + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m2 = ml_s[buf][nt * 4 + e][lane], l2 = ml_s[buf][nt * 4 + 2 + e][lane];
          const float mx = fmaxf(m_r[nt][e], m2);
          const float fa = m_r[nt][e] == mx ? 1.f : fast_exp2(m_r[nt][e] - mx), fb = m2 == mx ? 1.f : fast_exp2(m2 - mx);
          m_r[nt][e] = mx;
          l_r[nt][e] = l_r[nt][e] * fa + l2 * fb;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              o[mt][nt][e + 2 * h] = o[mt][nt][e + 2 * h] * fa + j[((mt * NT + nt) * 4 + e + 2 * h) * 32] * fb;
        }
    };
    if (warp & 1) put(warp >> 1);
    __syncthreads();
    if (!(warp & 1)) add(warp >> 1);
    if (warp == 2) put(1);
    __syncthreads();
    const long long unit_end = unit_begin + cu.T;
    const bool whole = unit_begin >= begin && unit_end <= end;
    const int dim0 = BITS == 8 ? 2 * g : 4 * g;
    auto store = [&](int mt, int nt, float (&acc)[4], const float (&inv)[2]) {
      const int dim = BITS == 8 ? 16 * mt + dim0 : 32 * (mt >> 1) + dim0 + 2 * (mt & 1);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * nt + 2 * q4 + e;
        if (row < rows)
          *reinterpret_cast<uint32_t*>(P.out + (size_t)(cu.t0 + row / G) * P.Hq * D + (size_t)(c_kvh * G + row % G) * D + dim) =
              pack_bf16(acc[e] * inv[e], acc[e + 2] * inv[e]);
      }
    };
    if (warp == 0) {
      add(1);
      if (whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float inv[2] = {1.f / l_r[nt][0], 1.f / l_r[nt][1]};
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) store(mt, nt, o[mt][nt], inv);
        }
      } else {
        float* seg_out = P.scratch + ((size_t)blockIdx.x * 2 + (begin >= unit_begin ? 0 : 1)) * C::kSegFloats;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            __stcg(reinterpret_cast<float4*>(seg_out) + (mt * NT + nt) * 32 + lane,
                   make_float4(o[mt][nt][0], o[mt][nt][1], o[mt][nt][2], o[mt][nt][3]));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          __stcg(reinterpret_cast<float4*>(seg_out) + (MT * NT + nt) * 32 + lane,
                 make_float4(m_r[nt][0], m_r[nt][1], l_r[nt][0], l_r[nt][1]));
      }
    }
    if (!whole) {
      // blocks whose share meets this unit: first .. last; the one that comes last joins them in order
      const int first = (int)(((unit_begin + 1) * nb - 1) / total), last = (int)((unit_end * nb - 1) / total);
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
        // warp w joins the row tiles mt = w, w + 4, ... of all segments
        auto seg_at = [&](int i) {
          const long long bi = total * i / nb;
          return reinterpret_cast<const float4*>(P.scratch + ((size_t)i * 2 + (bi >= unit_begin ? 0 : 1)) * C::kSegFloats) + lane;
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float mx[2] = {-INFINITY, -INFINITY}, ls[2] = {0.f, 0.f};
          float4 acc[MT / 4];
#pragma unroll
          for (int j = 0; j < MT / 4; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          constexpr int U = 8;
          for (int i0 = first; i0 <= last; i0 += U) {
            float4 ml[U], a[U][MT / 4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const float4* s = seg_at(min(i0 + u, last));
              ml[u] = __ldcg(s + (MT * NT + nt) * 32);
#pragma unroll
              for (int j = 0; j < MT / 4; ++j) a[u][j] = __ldcg(s + ((4 * j + warp) * NT + nt) * 32);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              if (i0 + u > last) break;
              const float m2[2] = {ml[u].x, ml[u].y}, l2[2] = {ml[u].z, ml[u].w};
              float fa[2], fb[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float m = fmaxf(mx[e], m2[e]);
                fa[e] = mx[e] == m ? 1.f : fast_exp2(mx[e] - m);
                fb[e] = m2[e] == m ? 1.f : fast_exp2(m2[e] - m);
                mx[e] = m;
                ls[e] = ls[e] * fa[e] + l2[e] * fb[e];
              }
#pragma unroll
              for (int j = 0; j < MT / 4; ++j) {
                acc[j].x = acc[j].x * fa[0] + a[u][j].x * fb[0];
                acc[j].y = acc[j].y * fa[1] + a[u][j].y * fb[1];
                acc[j].z = acc[j].z * fa[0] + a[u][j].z * fb[0];
                acc[j].w = acc[j].w * fa[1] + a[u][j].w * fb[1];
              }
            }
          }
          const float inv[2] = {1.f / ls[0], 1.f / ls[1]};
#pragma unroll
          for (int j = 0; j < MT / 4; ++j) {
            float r[4] = {acc[j].x, acc[j].y, acc[j].z, acc[j].w};
            store(4 * j + warp, nt, r, inv);
          }
        }
      }
    }
    // ---- on to the next unit
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
    }
  }
  if (absent_page || past_table) atomicOr(P.status, kStatusBadPage);
  if (lane == 0 && expired) atomicOr(P.status, kStatusWaitExpired);
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

// Query rows of a unit for up to `rows` (new tokens x heads of a group) rows a sequence.
static int row_tiles_of(int rows) { return rows <= 8 ? 1 : 2; }

}  // namespace siar

using namespace siar;

SIAR_DEFINE_PDL_SWITCH()

// 1 when the kernel takes these sizes (bfloat16 activations).
extern "C" int siar_attn_quant_supported(int Hq, int Hkv, int D, int page_tokens, long long n_pages) {
  if (Hkv <= 0 || Hq % Hkv != 0 || page_tokens <= 0) return 0;
  return (D == 64 || D == 128) && page_tokens % 64 == 0 && n_pages * Hkv * page_tokens < (1ll << 31);
}

// Blocks of a launch (the counters it needs); more never help: a block step is the least share.
extern "C" int siar_attn_quant_blocks(int B, int Hq, int Hkv, int D, int max_q_len, int max_kv_len, int sm_count) {
  const int rows = max_q_len * (Hq / Hkv), per_unit = 8 * row_tiles_of(rows);
  const int keys = D == 128 ? 128 : 256;
  const long long steps = (long long)B * Hkv * ((rows + per_unit - 1) / per_unit) * ((max_kv_len + keys - 1) / keys);
  return (int)(steps < 2ll * sm_count ? (steps > 0 ? steps : 1) : 2ll * sm_count);
}

// Scratch floats for that many blocks.
extern "C" long long siar_attn_quant_scratch_floats(int Hq, int Hkv, int D, int max_q_len, int blocks) {
  const int nt = row_tiles_of(max_q_len * (Hq / Hkv));
  return (long long)blocks * 2 * ((long long)(D / 16) * nt * 4 + 4 * nt) * 32;
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
// used.  counters: `blocks` zeros, left zero.
extern "C" int siar_attn_quant(int bits, const void* qkv, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                               const int* block_table, const int* slot_ids, const int* q_start, const int* base_len,
                               const float* inv_freq, void* out, float* scratch, int* counters, int blocks, int B, int Hq,
                               int Hkv, int D, int page_tokens, int max_pages, int n_pages, int max_q_len, int fused,
                               int write_kv, float scale, int* status, void* stream) {
  if (B == 0 || max_q_len == 0) return 0;
  if (!siar_attn_quant_supported(Hq, Hkv, D, page_tokens, n_pages) || (bits != 8 && bits != 4) || blocks <= 0 ||
      n_pages <= 0 || max_pages <= 0 || (long long)max_pages * page_tokens >= (1ll << 31) || (fused && max_q_len != 1))
    return (int)cudaErrorInvalidValue;
  QuantAttnParams p = {(const __nv_bfloat16*)qkv, (uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids,
                       q_start, base_len, inv_freq, (__nv_bfloat16*)out, scratch, counters, status, B, Hq, Hkv, page_tokens,
                       max_pages, n_pages, (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1, fused, write_kv, scale * 1.4426950408889634f};
  cudaStream_t s = (cudaStream_t)stream;
  const int nt = row_tiles_of(max_q_len * (Hq / Hkv));
#define SIAR_GO(BITS, DIM) \
  return nt == 1 ? launch_quant<BITS, DIM, 1>(p, blocks, s) : launch_quant<BITS, DIM, 2>(p, blocks, s)
  if (bits == 8) {
    if (D == 64) { SIAR_GO(8, 64); }
    SIAR_GO(8, 128);
  }
  if (D == 64) { SIAR_GO(4, 64); }
  SIAR_GO(4, 128);
#undef SIAR_GO
}
