// A key/value cache held in 8 or 4 bits: rotary encoding + quantisation of new tokens into the
// pages, and reading a batch's keys and values back as pages of the compute type.
//
// Formats (a row is one position of one kv head, D values x_0 .. x_{D-1}; keys are held rotated):
//   8 bits  codes int8 [pages][Hkv][page_tokens][D], scales float32 [pages][Hkv][page_tokens]
//           s = max|x| (1/127),  c_d = rint(x_d / s),  value c_d * s.   The reference's int8 cache has
//           the same row scale (model/kv_cache.py:58-67), rounded to 16 bits there, 32 here.
//   4 bits  codes uint8 [pages][Hkv][page_tokens][D/2] (dim 2i in the low half of byte i, 2i+1 in the
//           high half), scales bfloat16 [pages][Hkv][page_tokens][ceil(D/64)][2]: for every run of 64
//           dims s = bf16(max(x) (1/15) - min(x) (1/15)), m = bf16(min(x) + 8 s), c_d = rint((x_d - m) / s) + 8
//           within 0..15, value (c_d - 8) * s + m.  s and m are rounded to 16 bits because they are a
//           ninth of the format's bytes; the codes are taken against the rounded ones.  The scale is off by at most
//           2^-8 of itself, 15 * 2^-9 steps at the ends of the range.  The mid is off by at most 2^-8 of itself,
//           which for a run that lies far from zero beside its own range is many steps: of 100 and 100.5 (s = 0.0334,
//           m = 100.5 for 100.27) the lower one reads back as 100.23, seven steps off, its code at the end.
// A row (8 bits) or run (4 bits) that holds an infinity or a NaN gets the scale NaN and reads back as
// NaN: it is not turned into ordinary numbers.  A constant run has s = 0 and reads back as m.
//
// The rotation angle is position x frequency without rounding (a product of two 24-bit numbers fits a
// double), its cosine and sine are rounded to 32 bits once, and the rotated value is formed by two
// rounded products and a rounded sum, so a code depends on the token's row and position alone.
#include "kv_quant.cuh"

#include <cuda_fp16.h>

namespace siar {

// The batch description and the block table are read through plain pointers, behind pdl_wait(): the
// kernel in front may have written them (advance_lengths, set_table_cells), and a load through a
// const __restrict__ pointer may be moved in front of the wait.
__device__ __forceinline__ int sequence_of(const int* q_start, int B, int t) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q_start[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// ------------------------------------------------------------------ rotate, quantise, store
// grid (tokens, parts), 4 warps; the heads of a token (queries, keys, values) are dealt to the warps
// of its blocks.  A warp rotates its head into `row` (shared memory) and, for keys and values, takes
// scale and codes from there: lane l holds dims 64 i + 2l, + 2l + 1 of every run i, one byte of 4-bit
// codes or two of 8-bit codes.  Any head size in steps of 16 up to 256, any rotary layout.
template <typename T, int BITS>
__global__ void __launch_bounds__(128)
rope_quantize_kernel(const T* qkv, T* q_out, const float* __restrict__ inv_freq, uint8_t* __restrict__ k_pool,
                     uint8_t* __restrict__ v_pool, void* __restrict__ k_scale, void* __restrict__ v_scale,
                     const int* block_table, const int* slot_ids, const int* q_start, const int* base_len, int B, int Hq, int Hkv, int D,
                     int page_tokens, int max_pages, int n_pages, int write_kv, int* __restrict__ status,
                     int rotary_dim, int interleaved) {
  pdl_launch_dependents();
  __shared__ float cs[256];              // cos[half], sin[half]
  __shared__ float rows[4][256];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  if (t >= q_start[B]) return;           // a row behind the last sequence stays as it is
  const int b = sequence_of(q_start, B, t);
  const int pos = base_len[b] + (t - q_start[b]);
  const int half = rotary_dim >> 1;
  if (inv_freq != nullptr) {
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
      rotation(pos, inv_freq[i], &cs[i], &cs[half + i]);
    }
  }
  int page = -1;
  if (write_kv) {
    page = pos / page_tokens < max_pages ? block_table[(size_t)slot_ids[b] * max_pages + pos / page_tokens] : -1;
    if (page < 0 || page >= n_pages) {
      page = -1;
      if (threadIdx.x == 0) atomicOr(status, kStatusBadPage);
    }
  }
  __syncthreads();
  const size_t tok = (size_t)t * (Hq + 2 * Hkv) * D;
  const int heads = page >= 0 ? Hq + 2 * Hkv : Hq;
  float* row = rows[warp];
  for (int head = blockIdx.y * 4 + warp; head < heads; head += gridDim.y * 4) {
    const T* src = qkv + tok + (size_t)head * D;
    const bool rotates = inv_freq != nullptr && head < Hq + Hkv;
    __syncwarp();
    if (rotates) {
      for (int i = lane; i < half; i += 32) {
        const int i0 = interleaved ? 2 * i : i, i1 = interleaved ? 2 * i + 1 : i + half;
        const float a = to_f32(src[i0]), c = to_f32(src[i1]);
        row[i0] = rotate_lo(a, c, cs[i], cs[half + i]);
        row[i1] = rotate_hi(a, c, cs[i], cs[half + i]);
      }
    }
    for (int d = (rotates ? rotary_dim : 0) + lane; d < D; d += 32) row[d] = to_f32(src[d]);
    __syncwarp();
    if (head < Hq) {
      T* dst = q_out + tok + (size_t)head * D;
      for (int d = lane; d < D; d += 32) dst[d] = from_f32<T>(row[d]);
      continue;
    }
    const bool is_k = head < Hq + Hkv;
    const int kvh = is_k ? head - Hq : head - Hq - Hkv;
    const size_t at = ((size_t)page * Hkv + kvh) * page_tokens + pos % page_tokens;     // row of the pools
    uint8_t* codes = (is_k ? k_pool : v_pool) + at * (BITS == 8 ? D : D / 2);
    float* s8 = reinterpret_cast<float*>(is_k ? k_scale : v_scale) + at;
    __nv_bfloat162* s4 = reinterpret_cast<__nv_bfloat162*>(is_k ? k_scale : v_scale) + at * ((D + kQuantGroup - 1) / kQuantGroup);
    quantize_row<BITS>(
        row, D, lane,
        [&](int d, uint32_t c) {
          if (BITS == 8) *reinterpret_cast<uint16_t*>(codes + d) = (uint16_t)c;
          else codes[d / 2] = (uint8_t)c;
        },
        [&](int g, float s, __nv_bfloat162 sm) {
          if (BITS == 8) *s8 = s;
          else s4[g] = sm;
        });
  }
}

// The same for bfloat16, head_dim 64 or 128 and whole-head rotation in pairs (i, i + D/2), 16 bytes an access: D/16
// lanes share a head, a lane holds dims 8j .. 8j + 7 and D/2 + 8j .. + 7, so the pairs of a rotation are its own
// and a row's statistics take two or three shuffles.  A block walks a run of tokens, kTokens of them at a time:
// their sequences, pages and angles are formed together, and a token's heads are asked for while the token in
// front is worked on.  9,500 tokens of the 8B heads (8 bits): 43 us where their bytes take 34.  Instructions come next to
// memory as its bound: 8 bytes an access and a division for every code took 59 us (200 warp instructions for two
// heads), one token a block 61.
// F16: queries leave as float16 [tokens, Hq, D], each row times a power of two that brings its largest element to
// 2^9 .. 2^10, and that power's inverse as the row's factor (what the prompt attention on float16 tiles takes: 11 bits
// of a query where bfloat16 keeps 8).
template <int D, int BITS, bool F16>
__global__ void __launch_bounds__(128, 5)
rope_quantize_wide_kernel(const __nv_bfloat16* qkv, void* q_to, float* q_factor, const float* __restrict__ inv_freq,
                          uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, void* __restrict__ k_scale,
                          void* __restrict__ v_scale, const int* block_table, const int* slot_ids, const int* q_start,
                          const int* base_len, int N, int B, int Hq, int Hkv, int page_tokens, int max_pages, int n_pages,
                          int write_kv, int* __restrict__ status) {
  constexpr int LANES = D / 16, HEADS = 128 / LANES, kPasses = 3, NG = BITS == 8 ? 1 : D / kQuantGroup, kTokens = 4;
  pdl_launch_dependents();
  __shared__ __align__(16) float cos_s[kTokens][D / 2], sin_s[kTokens][D / 2];
  __shared__ int pos_s[kTokens], page_s[kTokens];
  const float freq = inv_freq != nullptr ? inv_freq[threadIdx.x % (D / 2)] : 0.f;
  pdl_wait();
  const int t_begin = (int)((long long)N * blockIdx.x / gridDim.x);
  int t_end = (int)((long long)N * (blockIdx.x + 1) / gridDim.x);
  const int lane = threadIdx.x & 31, j = threadIdx.x % LANES, h0 = threadIdx.x / LANES;
  const unsigned mates = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));       // the lanes that share the head
  const int heads = Hq + 2 * Hkv, stride = gridDim.y * HEADS;
  const size_t token_elems = (size_t)heads * D;
  uint4 lo[kPasses], hi[kPasses];
  auto load = [&](int t, int base) {                // kPasses heads of token t
    if (t >= t_end) return;
    const __nv_bfloat16* row = qkv + t * token_elems + (size_t)(base + h0) * D + 8 * j;
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
      if (base + h0 + p * stride < heads) {
        lo[p] = *reinterpret_cast<const uint4*>(row + (size_t)p * stride * D);
        hi[p] = *reinterpret_cast<const uint4*>(row + (size_t)p * stride * D + D / 2);
      }
  };
  load(t_begin, blockIdx.y * HEADS);
  const int used = q_start[B];                      // rows behind the last sequence stay as they are
  for (int t0 = t_begin; t0 < t_end; t0 += kTokens) {
    __syncthreads();                                // the angles of the tokens in front have been used
    if (threadIdx.x < 32) {
      // sequence of each token: for up to 32 sequences all of their descriptions are asked for at once
      const int t = t0 + lane;
      int pos = 0, slot = 0;
      if (B <= 32) {
        const int next = lane < B ? q_start[lane + 1] : 0x7fffffff, first = lane < B ? q_start[lane] : 0;
        const int base = lane < B ? base_len[lane] : 0, own = lane < B ? slot_ids[lane] : 0;
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
          const int b = min(__popc(__ballot_sync(0xffffffffu, next <= t0 + i)), B - 1);
          const int at = __shfl_sync(0xffffffffu, base - first, b), sl = __shfl_sync(0xffffffffu, own, b);
          if (lane == i) { pos = at + t; slot = sl; }
        }
      } else if (lane < kTokens && t < min(t_end, used)) {
        const int b = sequence_of(q_start, B, t);
        pos = base_len[b] + (t - q_start[b]);
        slot = slot_ids[b];
      }
      if (lane < kTokens && t < min(t_end, used)) {
        int page = -1;
        if (write_kv) {
          const int cell = pos / page_tokens;
          page = cell < max_pages ? block_table[(size_t)slot * max_pages + cell] : -1;
          if (page < 0 || page >= n_pages) {
            page = -1;
            atomicOr(status, kStatusBadPage);
          }
        }
        pos_s[lane] = pos;
        page_s[lane] = page;
      }
    }
    __syncthreads();
    t_end = min(t_end, used);                       // (here, where its load has come back)
    if (inv_freq != nullptr) {
      const int f = threadIdx.x % (D / 2);
      for (int i = threadIdx.x / (D / 2); i < kTokens && t0 + i < t_end; i += 128 / (D / 2))
        rotation(pos_s[i], freq, &cos_s[i][f], &sin_s[i][f]);
      __syncthreads();
    }
    for (int t = t0; t < min(t0 + kTokens, t_end); ++t) {
      const int page = page_s[t - t0];
      const size_t row0 = (size_t)max(page, 0) * Hkv * page_tokens + pos_s[t - t0] % page_tokens;      // kv head 0
      const float4* cs = reinterpret_cast<const float4*>(cos_s[t - t0]) + 2 * j;
      const float4* sn = reinterpret_cast<const float4*>(sin_s[t - t0]) + 2 * j;
      for (int base = blockIdx.y * HEADS; base < heads; base += kPasses * stride) {
        uint4 now_lo[kPasses], now_hi[kPasses];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          now_lo[p] = lo[p];
          now_hi[p] = hi[p];
        }
        if (base + kPasses * stride < heads) load(t, base + kPasses * stride);
        else load(t + 1, blockIdx.y * HEADS);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
          const int head = base + h0 + p * stride;
          if (head >= heads || (head >= Hq && page < 0)) continue;          // the same for all lanes of a head
          float x[16];
          const uint32_t w[8] = {now_lo[p].x, now_lo[p].y, now_lo[p].z, now_lo[p].w,
                                 now_hi[p].x, now_hi[p].y, now_hi[p].z, now_hi[p].w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
          if (inv_freq != nullptr && head < Hq + Hkv) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float4 c4 = cs[q], s4 = sn[q];
              const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float a = x[4 * q + e], c = x[8 + 4 * q + e];
                x[4 * q + e] = rotate_lo(a, c, cv[e], sv[e]);
                x[8 + 4 * q + e] = rotate_hi(a, c, cv[e], sv[e]);
              }
            }
          }
          if (head < Hq) {
            uint4 o[2];
            uint16_t* dst;
            if (F16) {
              float most = 0.f;
#pragma unroll
              for (int e = 0; e < 16; ++e) most = max_nan(most, fabsf(x[e]));
#pragma unroll
              for (int q = LANES / 2; q > 0; q >>= 1) most = max_nan(most, __shfl_xor_sync(mates, most, q));
              const int up = max(-120, min(60, 9 + 127 - (int)(__float_as_uint(most) >> 23)));
              const float f = __uint_as_float((uint32_t)(up + 127) << 23);
              __half2* o2 = reinterpret_cast<__half2*>(o);
#pragma unroll
              for (int e = 0; e < 8; ++e) o2[e] = __floats2half2_rn(x[2 * e] * f, x[2 * e + 1] * f);
              if (j == 0) q_factor[(size_t)t * Hq + head] = isfinite(most) ? 1.f / f : __int_as_float(0x7fc00000);
              dst = reinterpret_cast<uint16_t*>(q_to) + ((size_t)t * Hq + head) * D + 8 * j;
            } else {
              __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(o);
#pragma unroll
              for (int e = 0; e < 8; ++e) o2[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
              dst = reinterpret_cast<uint16_t*>(q_to) + t * token_elems + (size_t)head * D + 8 * j;
            }
            *reinterpret_cast<uint4*>(dst) = o[0];
            *reinterpret_cast<uint4*>(dst + D / 2) = o[1];
            continue;
          }
          const bool is_k = head < Hq + Hkv;
          const size_t at = row0 + (size_t)(is_k ? head - Hq : head - Hq - Hkv) * page_tokens;
          uint8_t* codes = (is_k ? k_pool : v_pool) + at * (D * BITS / 8);
          // largest and smallest of a run (8 bits: largest |x| of the row); NaN if one is
          constexpr int PER = 16 / NG;
          float top[NG], bot[NG];
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float most = -INFINITY, least = -INFINITY;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              const float y = x[g * PER + e];
              most = max_nan(most, BITS == 8 ? fabsf(y) : y);
              if (BITS == 4) least = max_nan(least, -y);
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) {
              most = max_nan(most, __shfl_xor_sync(mates, most, o));
              if (BITS == 4) least = max_nan(least, __shfl_xor_sync(mates, least, o));
            }
            top[g] = most;
            bot[g] = -least;
          }
          if (BITS == 8) {
            const float s = scale8(top[0]);
            const bool bad = !isfinite(top[0]);
            const Divisor by = divisor(s);
            if (by.k != 1.f) {                      // (a scale near the ends of the range may itself be rounded coarsely)
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = fmaxf(-127.f * by.s, fminf(127.f * by.s, x[e] * by.k));
            }
            uint32_t c[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) c[e] = whole_bits(corrected(x[e], by));       // |x| <= 127 s (1 + 2^-23): no code leaves its byte
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              b[e] = __byte_perm(__byte_perm(c[4 * e], c[4 * e + 1], 0x0040), __byte_perm(c[4 * e + 2], c[4 * e + 3], 0x0040), 0x5410);
            *reinterpret_cast<uint2*>(codes + 8 * j) = bad ? make_uint2(0u, 0u) : make_uint2(b[0], b[1]);
            *reinterpret_cast<uint2*>(codes + D / 2 + 8 * j) = bad ? make_uint2(0u, 0u) : make_uint2(b[2], b[3]);
            if (j == 0) reinterpret_cast<float*>(is_k ? k_scale : v_scale)[at] = bad ? __int_as_float(0x7fc00000) : s;
          } else {
            __nv_bfloat162* sc = reinterpret_cast<__nv_bfloat162*>(is_k ? k_scale : v_scale) + at * NG;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int g = NG == 1 ? 0 : h;
              const bool bad = !isfinite(top[g]) || !isfinite(bot[g]);
              const __nv_bfloat162 sm = scale4(bot[g], top[g], bad);
              const Divisor by = divisor(__low2float(sm));
              const float m = __high2float(sm);
              uint32_t c = 0;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float y = __fsub_rn(x[8 * h + e], m);
                if (by.k != 1.f) y *= by.k;
                c |= ((whole_bits(fmaxf(-8.f, fminf(7.f, corrected(y, by)))) + 8u) & 15u) << (4 * e);
              }
              *reinterpret_cast<uint32_t*>(codes + h * (D / 4) + 4 * j) = bad ? 0x88888888u : c;
              if (j == 0 && (NG == 2 || h == 0)) sc[g] = sm;
            }
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------ read back
// Sequence b's pages go, in order, behind those of the sequences before it: page p of sequence b is
// page first(b) + p of the output pools [pages][Hkv][page_tokens][D]; row b of `out_table` names them
// (-1 beyond), `out_slots[b]` = b (nullptr: not written).  Rows behind a sequence's last token are zeros.  Pages that lie
// wholly in front of every query's window (first_key of the batch's first new token) are not read.
// grid (pages of the longest sequence, Hkv, B), 256 threads, 16 codes a thread and step.  Memory bounds it: 9,500 tokens of
// the 8B heads in 8 bits 16 us where the bytes take 9 (four steps asked for together: 19, fewer blocks fit an SM).
template <typename T, int BITS>
__global__ void __launch_bounds__(256)
read_kv_kernel(const uint8_t* k_pool, const uint8_t* v_pool, const void* k_scale, const void* v_scale,
               const int* block_table, const int* slot_ids, const int* q_start, const int* base_len, T* __restrict__ k_out, T* __restrict__ v_out,
               int* __restrict__ out_table, int* __restrict__ out_slots, int B, int Hkv, int D, int page_tokens,
               int max_pages, int n_pages, int pages_out, int max_kv_len, int window, int* __restrict__ status) {
  pdl_launch_dependents();
  __shared__ int first_s;
  pdl_wait();
  const int p = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int most = min((max_kv_len + page_tokens - 1) / page_tokens, max_pages);
  auto pages_of = [&](int i) {
    return min((base_len[i] + q_start[i + 1] - q_start[i] + page_tokens - 1) / page_tokens, most);
  };
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int i = threadIdx.x; i < b; i += 32) sum += pages_of(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) first_s = sum;
  }
  __syncthreads();
  const int first = first_s, mine = pages_of(b);
  const int total = base_len[b] + q_start[b + 1] - q_start[b];
  const int unseen = window > 0 ? max(0, base_len[b] - window + 1) / page_tokens : 0;     // pages nobody looks at
  if (p == 0 && kvh == 0) {
    for (int i = threadIdx.x; i < max_pages; i += blockDim.x)
      out_table[(size_t)b * max_pages + i] = i >= unseen && i < mine && first + i < pages_out ? first + i : -1;
    if (threadIdx.x == 0) {
      if (out_slots != nullptr) out_slots[b] = b;
      if ((total + page_tokens - 1) / page_tokens > most) atomicOr(status, kStatusLengthPastGrid);
    }
  }
  if (p >= mine || p < unseen || first + p >= pages_out) return;
  int page = block_table[(size_t)slot_ids[b] * max_pages + p];
  const bool absent = page < 0 || page >= n_pages;
  if (absent) {
    page = 0;
    if (threadIdx.x == 0) atomicOr(status, kStatusBadPage);
  }
  const size_t row0 = ((size_t)page * Hkv + kvh) * page_tokens;
  const size_t out0 = ((size_t)(first + p) * Hkv + kvh) * page_tokens;
  const int rows_held = absent ? 0 : min(page_tokens, total - p * page_tokens);
  const int per_row = D / 16, groups = (D + kQuantGroup - 1) / kQuantGroup;
  for (int idx = threadIdx.x; idx < 2 * page_tokens * per_row; idx += blockDim.x) {
    const bool is_k = idx < page_tokens * per_row;
    const int i = is_k ? idx : idx - page_tokens * per_row;
    const int r = i / per_row, d = (i % per_row) * 16;
    // a code as a float: its bits in the mantissa of 2^23, the constant taken off again (both exact); 4-bit codes stand for
    // code - 8
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
    if (r < rows_held) {
      const uint8_t* src = (is_k ? k_pool : v_pool) + ((row0 + r) * D + d) * BITS / 8;
      const uint32_t* sc = reinterpret_cast<const uint32_t*>(is_k ? k_scale : v_scale);
      if (BITS == 8) {
        const uint4 code = *reinterpret_cast<const uint4*>(src);
        const uint32_t w[4] = {code.x, code.y, code.z, code.w};
        const float s = __uint_as_float(sc[row0 + r]);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = (__uint_as_float(__byte_perm(w[e >> 2] ^ 0x80808080u, 0x4b000000u, 0x7440 + (e & 3))) - 8388736.f) * s;
      } else {
        const uint2 code = *reinterpret_cast<const uint2*>(src);
        const uint32_t w[2] = {code.x, code.y}, at = sc[(row0 + r) * groups + d / kQuantGroup];
        const float s = __uint_as_float(at << 16), m = __uint_as_float(at & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = __fadd_rn(__fmul_rn(__uint_as_float(((w[e >> 3] >> (4 * (e & 7))) & 15u) | 0x4b000000u) - 8388616.f, s), m);
      }
    }
    T* dst = (is_k ? k_out : v_out) + (out0 + r) * D + d;
    if (sizeof(T) == 2) {
      uint4 pk[2];
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(pk);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      reinterpret_cast<uint4*>(dst)[0] = pk[0];
      reinterpret_cast<uint4*>(dst)[1] = pk[1];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<float4*>(dst)[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    }
  }
}

}  // namespace siar

using namespace siar;

SIAR_DEFINE_PDL_SWITCH()

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  return n;
}

template <bool F16>
static int launch_wide(int bits, const void* qkv, void* q_to, float* q_factor, const float* inv_freq, void* k_pool, void* v_pool,
                       void* k_scale, void* v_scale, const int* block_table, const int* slot_ids, const int* q_start,
                       const int* base_len, int N, int B, int Hq, int Hkv, int D, int page_tokens, int max_pages, int n_pages,
                       int write_kv, int* status, void* stream) {
  const int per_block = 128 / (D / 16);             // few tokens: the heads of one token go to several blocks
  const int most = (Hq + 2 * Hkv + per_block - 1) / per_block, split = N >= 296 ? 1 : min(most, (296 + N - 1) / N);
  const int blocks = min(N, 5 * sm_count());
  auto go = [&](auto kernel) {
    return (int)launch_kernel(kernel, dim3(blocks, split), dim3(128), 0, (cudaStream_t)stream, (const __nv_bfloat16*)qkv, q_to,
                              q_factor, inv_freq, (uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids,
                              q_start, base_len, N, B, Hq, Hkv, page_tokens, max_pages, n_pages, write_kv, status);
  };
  if (bits == 8) return D == 64 ? go(rope_quantize_wide_kernel<64, 8, F16>) : go(rope_quantize_wide_kernel<128, 8, F16>);
  return D == 64 ? go(rope_quantize_wide_kernel<64, 4, F16>) : go(rope_quantize_wide_kernel<128, 4, F16>);
}

// qkv [N, (Hq + 2 Hkv) D] (not changed unless q_out == qkv); q_out: the same layout, its query part is
// written (rotated).  Pools and scales as at the top of the file.
static int siar_rope_quantize_of(int is_bf16, int bits, const void* qkv, void* q_out, const float* inv_freq,
                                  void* k_pool, void* v_pool, void* k_scale, void* v_scale, const int* block_table,
                                  const int* slot_ids, const int* q_start, const int* base_len, int N, int B, int Hq,
                                  int Hkv, int D, int page_tokens, int max_pages, int n_pages, int write_kv,
                                  int* status, void* stream, int rotary_dim, int interleaved) {
  if (N == 0) return 0;
  if ((bits != 8 && bits != 4) || D % 16 != 0 || D <= 0 || D > 256 || rotary_dim < 0 || rotary_dim > D ||
      rotary_dim % 2 != 0 || page_tokens <= 0)
    return (int)cudaErrorInvalidValue;
  if (is_bf16 && (D == 64 || D == 128) && (inv_freq == nullptr || (rotary_dim == D && !interleaved)) &&
      (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0)
    return launch_wide<false>(bits, qkv, q_out, nullptr, inv_freq, k_pool, v_pool, k_scale, v_scale, block_table, slot_ids, q_start,
                              base_len, N, B, Hq, Hkv, D, page_tokens, max_pages, n_pages, write_kv, status, stream);
  // few tokens: the heads of one token go to several blocks
  const int parts = N >= 592 ? 1 : min((Hq + 2 * Hkv + 3) / 4, (592 + N - 1) / N);
  auto go = [&](auto kernel, auto* typed) {
    using T = typename std::remove_pointer<decltype(typed)>::type;
    return (int)launch_kernel(kernel, dim3(N, parts), dim3(128), 0, (cudaStream_t)stream, (const T*)qkv, (T*)q_out, inv_freq,
                              (uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids, q_start,
                              base_len, B, Hq, Hkv, D, page_tokens, max_pages, n_pages, write_kv, status, rotary_dim,
                              interleaved);
  };
  if (is_bf16)
    return bits == 8 ? go(rope_quantize_kernel<__nv_bfloat16, 8>, (__nv_bfloat16*)nullptr)
                     : go(rope_quantize_kernel<__nv_bfloat16, 4>, (__nv_bfloat16*)nullptr);
  return bits == 8 ? go(rope_quantize_kernel<float, 8>, (float*)nullptr)
                   : go(rope_quantize_kernel<float, 4>, (float*)nullptr);
}
SIAR_TAKES_WORDS(siar_rope_quantize)

// The same for bfloat16, head_dim 64 or 128 and whole-head rotation (or none), with the queries as float16:
// q16 [N, Hq, D], q_factor [N, Hq].
static int siar_rope_quantize_q16_of(int bits, const void* qkv, void* q16, float* q_factor, const float* inv_freq, void* k_pool,
                                      void* v_pool, void* k_scale, void* v_scale, const int* block_table, const int* slot_ids,
                                      const int* q_start, const int* base_len, int N, int B, int Hq, int Hkv, int D, int page_tokens,
                                      int max_pages, int n_pages, int write_kv, int* status, void* stream) {
  if (N == 0) return 0;
  if ((bits != 8 && bits != 4) || (D != 64 && D != 128) || page_tokens <= 0 ||
      (((uintptr_t)qkv | (uintptr_t)q16 | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0)
    return (int)cudaErrorInvalidValue;
  return launch_wide<true>(bits, qkv, q16, q_factor, inv_freq, k_pool, v_pool, k_scale, v_scale, block_table, slot_ids, q_start,
                           base_len, N, B, Hq, Hkv, D, page_tokens, max_pages, n_pages, write_kv, status, stream);
}
SIAR_TAKES_WORDS(siar_rope_quantize_q16)

// The keys and values of a batch as pages of the compute type; see read_kv_kernel.  out_table
// [B, max_pages], out_slots [B]; pages_out: pages the output pools have (host lengths that fall short of
// the device's leave the pages beyond unread, with cell -1).
static int siar_read_kv_of(int is_bf16, int bits, const void* k_pool, const void* v_pool, const void* k_scale,
                            const void* v_scale, const int* block_table, const int* slot_ids, const int* q_start,
                            const int* base_len, void* k_out, void* v_out, int* out_table, int* out_slots, int B,
                            int Hkv, int D, int page_tokens, int max_pages, int n_pages, int pages_out, int max_kv_len,
                            int window, int* status, void* stream) {
  if (B == 0) return 0;
  if ((bits != 8 && bits != 4) || D % 16 != 0 || D <= 0 || D > 256 || B > 65535 || Hkv > 65535 || page_tokens <= 0 ||
      max_kv_len <= 0)
    return (int)cudaErrorInvalidValue;
  const int pages = (max_kv_len + page_tokens - 1) / page_tokens;
  auto go = [&](auto kernel, auto* typed) {
    using T = typename std::remove_pointer<decltype(typed)>::type;
    return (int)launch_kernel(kernel, dim3(pages, Hkv, B), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)k_pool,
                              (const uint8_t*)v_pool, k_scale, v_scale, block_table, slot_ids, q_start, base_len,
                              (T*)k_out, (T*)v_out, out_table, out_slots, B, Hkv, D, page_tokens, max_pages, n_pages,
                              pages_out, max_kv_len, window, status);
  };
  if (is_bf16)
    return bits == 8 ? go(read_kv_kernel<__nv_bfloat16, 8>, (__nv_bfloat16*)nullptr)
                     : go(read_kv_kernel<__nv_bfloat16, 4>, (__nv_bfloat16*)nullptr);
  return bits == 8 ? go(read_kv_kernel<float, 8>, (float*)nullptr) : go(read_kv_kernel<float, 4>, (float*)nullptr);
}
SIAR_TAKES_WORDS(siar_read_kv)
