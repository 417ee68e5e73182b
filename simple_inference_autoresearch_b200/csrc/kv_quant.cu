// A key/value cache held in 8 or 4 bits: rotary encoding + quantisation of new tokens into the
// pages, and reading a batch's keys and values back as pages of the compute type.
//
// Formats (a row is one position of one kv head, D values x_0 .. x_{D-1}; keys are held rotated):
//   8 bits  codes int8 [pages][Hkv][page_tokens][D], scales float32 [pages][Hkv][page_tokens]
//           s = max|x| / 127,  c_d = rint(x_d / s),  value c_d * s.   The reference's int8 cache has
//           the same row scale (model/kv_cache.py:58-67), rounded to 16 bits there, 32 here.
//   4 bits  codes uint8 [pages][Hkv][page_tokens][D/2] (dim 2i in the low half of byte i, 2i+1 in the
//           high half), scales bfloat16 [pages][Hkv][page_tokens][ceil(D/64)][2]: for every run of 64
//           dims s = bf16(max(x)/15 - min(x)/15), m = bf16(min(x) + 8 s), c_d = rint((x_d - m) / s) + 8
//           within 0..15, value (c_d - 8) * s + m.  s and m are rounded to 16 bits because they are a
//           ninth of the format's bytes; the codes are taken against the rounded ones, so that costs
//           at most 15 * 2^-9 steps at the ends of the range.
// A row (8 bits) or run (4 bits) that holds an infinity or a NaN gets the scale NaN and reads back as
// NaN: it is not turned into ordinary numbers.  A constant run has s = 0 and reads back as m.
//
// The rotation angle is position x frequency without rounding (a product of two 24-bit numbers fits a
// double), its cosine and sine are rounded to 32 bits once, and the rotated value is formed by two
// rounded products and a rounded sum, so a code depends on the token's row and position alone.
#include "kv_quant.cuh"

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

// The same for bfloat16, head_dim 64 or 128 and whole-head rotation in pairs (i, i + D/2), 8 bytes an access: D/8
// lanes share a head, a lane holds dims 4j .. 4j + 3 and D/2 + 4j .. + 3, so the pairs of a rotation are its own
// and a row's statistics take a few shuffles.  A block of 256 threads takes a token's heads kPasses x 256 / (D/8)
// at a time, all of their loads asked for before the rotation angles are formed.
template <int D, int BITS>
__global__ void __launch_bounds__(256)
rope_quantize_wide_kernel(const __nv_bfloat16* qkv, __nv_bfloat16* q_out, const float* __restrict__ inv_freq,
                          uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, void* __restrict__ k_scale,
                          void* __restrict__ v_scale, const int* block_table, const int* slot_ids, const int* q_start,
                          const int* base_len, int B, int Hq, int Hkv, int page_tokens, int max_pages, int n_pages,
                          int write_kv, int* __restrict__ status) {
  constexpr int LANES = D / 8, HEADS = 256 / LANES, kPasses = 3, NG = D / kQuantGroup;
  pdl_launch_dependents();
  __shared__ float cos_s[D / 2], sin_s[D / 2];
  float freq = 0.f;
  if (inv_freq != nullptr && threadIdx.x < D / 2) freq = inv_freq[threadIdx.x];
  pdl_wait();
  const int t = blockIdx.x;
  const int j = threadIdx.x % LANES, h0 = threadIdx.x / LANES;
  const int heads = Hq + 2 * Hkv, stride = gridDim.y * HEADS;
  const __nv_bfloat16* row = qkv + (size_t)t * heads * D + 4 * j;
  uint2 lo[kPasses], hi[kPasses];
  auto load = [&](int first) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int head = first + p * stride;
      if (head < heads) {
        lo[p] = *reinterpret_cast<const uint2*>(row + (size_t)head * D);
        hi[p] = *reinterpret_cast<const uint2*>(row + (size_t)head * D + D / 2);
      }
    }
  };
  int first = blockIdx.y * HEADS + h0;
  load(first);
  const int b = sequence_of(q_start, B, t);
  const int pos = base_len[b] + (t - q_start[b]);
  if (inv_freq != nullptr && threadIdx.x < D / 2) rotation(pos, freq, &cos_s[threadIdx.x], &sin_s[threadIdx.x]);
  int page = -1;
  if (write_kv) {
    page = pos / page_tokens < max_pages ? block_table[(size_t)slot_ids[b] * max_pages + pos / page_tokens] : -1;
    if (page < 0 || page >= n_pages) {
      page = -1;
      if (threadIdx.x == 0) atomicOr(status, kStatusBadPage);
    }
  }
  __syncthreads();
  const size_t row0 = (size_t)max(page, 0) * Hkv * page_tokens + pos % page_tokens;      // kv head 0
  float cv[4], sv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cv[e] = inv_freq != nullptr ? cos_s[4 * j + e] : 1.f;
    sv[e] = inv_freq != nullptr ? sin_s[4 * j + e] : 0.f;
  }
  // of the lanes that share a head
  auto group_max = [](float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  // every thread runs every round: the shuffles take whole warps
  for (int base = blockIdx.y * HEADS; base < heads; base += kPasses * stride) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int head = base + h0 + p * stride;
      if (base + p * stride >= heads) break;
      const bool in = head < heads;
      float x[8];
      const uint2 l = in ? lo[p] : make_uint2(0u, 0u), u = in ? hi[p] : make_uint2(0u, 0u);
      const uint32_t w[4] = {l.x, l.y, u.x, u.y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(w[e] << 16);
        x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
      if (inv_freq != nullptr && head < Hq + Hkv) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = x[e], c = x[4 + e];
          x[e] = rotate_lo(a, c, cv[e], sv[e]);
          x[4 + e] = rotate_hi(a, c, cv[e], sv[e]);
        }
      }
      if (in && head < Hq) {
        __nv_bfloat16* dst = q_out + (size_t)t * heads * D + (size_t)head * D + 4 * j;
        uint2 o[2];
        __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(o);
#pragma unroll
        for (int e = 0; e < 4; ++e) o2[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<uint2*>(dst) = o[0];
        *reinterpret_cast<uint2*>(dst + D / 2) = o[1];
      }
      // (lanes of query heads in a warp with key heads go along for the shuffles)
      const bool is_k = head < Hq + Hkv, stores = in && head >= Hq && page >= 0;
      if (!__any_sync(0xffffffffu, stores)) continue;
      const int kvh = is_k ? head - Hq : head - Hq - Hkv;
      const size_t at = row0 + (size_t)max(kvh, 0) * page_tokens;
      uint8_t* codes = (is_k ? k_pool : v_pool) + at * (D * BITS / 8);
      float top[NG], bot[NG];                       // per run (8 bits: per row, of |x|)
      bool bad[NG];
      if (BITS == 8 || NG == 1) {
        float m = 0.f, n = INFINITY, a = -INFINITY;
        bool wrong = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m = fmaxf(m, fabsf(x[e]));
          n = fminf(n, x[e]);
          a = fmaxf(a, x[e]);
          wrong |= !isfinite(x[e]);
        }
        top[0] = group_max(BITS == 8 ? m : a);
        bot[0] = BITS == 8 ? 0.f : -group_max(-n);
        bad[0] = group_max(wrong ? 1.f : 0.f) > 0.f;
      } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float* y = x + 4 * g;
          const bool wrong = !isfinite(y[0]) || !isfinite(y[1]) || !isfinite(y[2]) || !isfinite(y[3]);
          top[g] = group_max(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
          bot[g] = -group_max(-fminf(fminf(y[0], y[1]), fminf(y[2], y[3])));
          bad[g] = group_max(wrong ? 1.f : 0.f) > 0.f;
        }
      }
      if (!stores) continue;
      if (BITS == 8) {
        const float s = scale8(top[0]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t c = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) c |= (uint32_t)(code8(x[4 * h + e], s, bad[0]) & 0xff) << (8 * e);
          *reinterpret_cast<uint32_t*>(codes + h * (D / 2) + 4 * j) = c;
        }
        if (j == 0) reinterpret_cast<float*>(is_k ? k_scale : v_scale)[at] = bad[0] ? __int_as_float(0x7fc00000) : s;
      } else {
        __nv_bfloat162* sc = reinterpret_cast<__nv_bfloat162*>(is_k ? k_scale : v_scale) + at * NG;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int g = NG == 1 ? 0 : h;
          const __nv_bfloat162 sm = scale4(bot[g], top[g], bad[g]);
          const float s = __low2float(sm), m = __high2float(sm);
          uint32_t c = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) c |= (uint32_t)code4(x[4 * h + e], s, m) << (4 * e);
          *reinterpret_cast<uint16_t*>(codes + h * (D / 4) + 2 * j) = (uint16_t)c;
          if (j == 0 && (NG == 2 || h == 0)) sc[g] = sm;
        }
      }
    }
    first += kPasses * stride;
    load(first);
  }
}

// ------------------------------------------------------------------ read back
// Sequence b's pages go, in order, behind those of the sequences before it: page p of sequence b is
// page first(b) + p of the output pools [pages][Hkv][page_tokens][D]; row b of `out_table` names them
// (-1 beyond), `out_slots[b]` = b.  Rows behind a sequence's last token are zeros.  Pages that lie
// wholly in front of every query's window (first_key of the batch's first new token) are not read.
// grid (pages of the longest sequence, Hkv, B), 256 threads, 16 codes a thread and step.
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
      out_slots[b] = b;
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
    float x[16];
    if (r >= rows_held) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
    } else if (BITS == 8) {
      const float s = reinterpret_cast<const float*>(is_k ? k_scale : v_scale)[row0 + r];
      const int4 c = *reinterpret_cast<const int4*>((is_k ? k_pool : v_pool) + (row0 + r) * D + d);
      const int w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * s;
    } else {
      const __nv_bfloat162 sm = reinterpret_cast<const __nv_bfloat162*>(is_k ? k_scale : v_scale)[(row0 + r) * groups + d / kQuantGroup];
      const float s = __low2float(sm), m = __high2float(sm);
      const int2 c = *reinterpret_cast<const int2*>((is_k ? k_pool : v_pool) + ((row0 + r) * D + d) / 2);
      const int w[2] = {c.x, c.y};
#pragma unroll
      for (int e = 0; e < 16; ++e)
        x[e] = __fadd_rn(__fmul_rn((float)(((w[e >> 3] >> (4 * (e & 7))) & 15) - 8), s), m);
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

// qkv [N, (Hq + 2 Hkv) D] (not changed unless q_out == qkv); q_out: the same layout, its query part is
// written (rotated).  Pools and scales as at the top of the file.
extern "C" int siar_rope_quantize(int is_bf16, int bits, const void* qkv, void* q_out, const float* inv_freq,
                                  void* k_pool, void* v_pool, void* k_scale, void* v_scale, const int* block_table,
                                  const int* slot_ids, const int* q_start, const int* base_len, int N, int B, int Hq,
                                  int Hkv, int D, int page_tokens, int max_pages, int n_pages, int write_kv,
                                  int* status, void* stream, int rotary_dim, int interleaved) {
  if (N == 0) return 0;
  if ((bits != 8 && bits != 4) || D % 16 != 0 || D <= 0 || D > 256 || rotary_dim < 0 || rotary_dim > D ||
      rotary_dim % 2 != 0 || page_tokens <= 0)
    return (int)cudaErrorInvalidValue;
  if (is_bf16 && (D == 64 || D == 128) && (inv_freq == nullptr || (rotary_dim == D && !interleaved)) &&
      (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0) {
    const int per_block = 256 / (D / 8);            // few tokens: the heads of one token go to several blocks
    const int most = (Hq + 2 * Hkv + per_block - 1) / per_block, split = N >= 296 ? 1 : min(most, (296 + N - 1) / N);
    auto wide = [&](auto kernel) {
      return (int)launch_kernel(kernel, dim3(N, split), dim3(256), 0, (cudaStream_t)stream, (const __nv_bfloat16*)qkv,
                                (__nv_bfloat16*)q_out, inv_freq, (uint8_t*)k_pool, (uint8_t*)v_pool, k_scale, v_scale,
                                block_table, slot_ids, q_start, base_len, B, Hq, Hkv, page_tokens, max_pages, n_pages, write_kv,
                                status);
    };
    if (bits == 8) return D == 64 ? wide(rope_quantize_wide_kernel<64, 8>) : wide(rope_quantize_wide_kernel<128, 8>);
    return D == 64 ? wide(rope_quantize_wide_kernel<64, 4>) : wide(rope_quantize_wide_kernel<128, 4>);
  }
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

// The keys and values of a batch as pages of the compute type; see read_kv_kernel.  out_table
// [B, max_pages], out_slots [B]; pages_out: pages the output pools have (host lengths that fall short of
// the device's leave the pages beyond unread, with cell -1).
extern "C" int siar_read_kv(int is_bf16, int bits, const void* k_pool, const void* v_pool, const void* k_scale,
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
