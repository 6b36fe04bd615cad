// Attention over a paged cache that is held in 8 bits: the formulas, the tables and the mask of attention.hip (causal, window,
// sink), over keys and values that stand for e4m3(code) * scale with one scale, a power of two, for the keys and one for the values
// of every (page, kv head). Codes [pages, Hkv, page_size, D], scales float32 [pages, Hkv].
//
// e4m3 times a power of two is a bfloat16 number as it is: the matrix-core kernels below turn codes into bfloat16 with the scale in
// the converting instruction and lose nothing there.
#include "attention.h"
#include "common.h"
#include "device.h"
#include "mfma.h"
#include <math.h>
#include <type_traits>

// What all kernels here are given.
struct F8Cache {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
};
struct F8Tables {
  const int32_t *q_start, *ctx_len, *block_table;
  int bt_stride;
};

// ===========================================================================
// ptl_attention_generic_f8: float32 arithmetic on the vector units, for every type of query, head size (up to 640), page size
// and number of heads. A workgroup has one query row of one head; its waves take the keys 64 at a time in turn, a lane a key
// for the scores (rows of a multiple of 16 elements by 16 bytes) and a lane every 64th column for the values, of which a wave asks for AHEAD
// rows before it uses one: with one at a time a turn was 64 ways to memory. Few rows have sixteen waves, more than two a compute unit
// four: us with sixteen and four, float32, 32 heads of 64 on 8: 32 x 2,000 keys 82 45, 64 x 100 to 1,000 113 31, 60 rows behind 300 42 16,
// 200 behind 700 153 71.
//
// What bounds it: few rows the chain of a turn, some 3 us (1 x 1,000 keys 7.8 us, 1 x 4,000 18.3, 8 x 2,048 27.2), many the vector units, which
// have every key row anew for every query row (200 rows behind 700: 19 TFLOP/s).
template <typename T, int NACC, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
attn_generic_f8_kernel(T* __restrict__ out, long out_stride, const T* __restrict__ q, long q_stride, F8Cache cache, F8Tables tab,
                       const int32_t* __restrict__ work_seq, const int32_t* __restrict__ work_qoff, int Hq, int Hkv, int D,
                       int page_size, int window, const float* __restrict__ sink, float scale) {
  constexpr int AHEAD = NACC <= 2 ? 16 : NACC <= 4 ? 8 : 4, THREADS = 64 * WAVES;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float ps[WAVES][64];          // a tile's probabilities times the values' scales
  __shared__ long at[WAVES][64];           // where its value rows lie
  __shared__ float ends[WAVES][2];
  float* qs = lds;                         // [D]
  float* sums = lds + D;                   // [WAVES][D]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // heads run fastest over the workgroups, which the eight dies take in turn: die c gets heads c Hq / 8 .. of which a kv head's lie together
  // (rows fastest, the first rows of blocks, decoding requests', would all be one die's)
  const int place = blockIdx.x / Hq, i_head = blockIdx.x - place * Hq;
  const int item = place >> 4, head = Hq % 8 == 0 ? (i_head % 8) * (Hq / 8) + i_head / 8 : i_head;
  const int seq = work_seq[item], r = work_qoff[item] + (place & 15);
  const int first = tab.q_start[seq], rows = tab.q_start[seq + 1] - first, ctx = tab.ctx_len[seq];
  if (r >= rows) return;
  const int row = first + r, pos = ctx - rows + r, kvh = head / (Hq / Hkv);
  const int32_t* bt = tab.block_table + (size_t)seq * tab.bt_stride;
  for (int d = threadIdx.x; d < D; d += THREADS) qs[d] = to_float<T>(q[(size_t)row * q_stride + (size_t)head * D + d]);
  __syncthreads();
  const int lo = window > 0 ? max(0, pos - window + 1) : 0;
  float m = -INFINITY, l = 0.f, acc[NACC];
#pragma unroll
  for (int a = 0; a < NACC; ++a) acc[a] = 0.f;
  auto four = [&](uint32_t x, const float* y, float dot) __attribute__((always_inline)) {
    const auto e = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), f = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
    return fmaf(f[1], y[3], fmaf(f[0], y[2], fmaf(e[1], y[1], fmaf(e[0], y[0], dot))));
  };
  for (int k0 = lo + 64 * wave; k0 <= pos; k0 += THREADS) {
    const int n = min(64, pos + 1 - k0), key = k0 + min(lane, n - 1);        // (lanes behind the last key: that one, weight zero)
    const int slot = key / page_size, page = bt[slot];
    const size_t block = (size_t)page * Hkv + kvh;
    const long row_at = (block * page_size + (key - slot * page_size)) * D;
    const float ks = cache.k_scale[block], vs = cache.v_scale[block];
    const uint8_t* kr = cache.k + row_at;
    float dot = 0.f;
    if (D % 16 == 0) {
#pragma unroll 4
      for (int d = 0; d < D; d += 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(kr + d);
        dot = four(x.w, qs + d + 12, four(x.z, qs + d + 8, four(x.y, qs + d + 4, four(x.x, qs + d, dot))));
      }
    } else if (D % 4 == 0) {
#pragma unroll 8
      for (int d = 0; d < D; d += 4) dot = four(*reinterpret_cast<const uint32_t*>(kr + d), qs + d, dot);
    } else {
#pragma unroll 8
      for (int d = 0; d < D; ++d) dot = fmaf(__builtin_amdgcn_cvt_f32_fp8((int)kr[d], 0), qs[d], dot);
    }
    const float s = lane < n ? dot * ks * scale : -INFINITY;
    const float top = fmaxf(m, wave_max(s));
    const float to = top == -INFINITY ? 0.f : top, keep = expf(m - to);
    const float p = lane < n ? expf(s - to) : 0.f;
    l = l * keep + wave_sum(p);
    m = top;
    ps[wave][lane] = p * vs;
    at[wave][lane] = row_at;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");       // (a wave's own LDS: written above, read below)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int a = 0; a < NACC; ++a) acc[a] *= keep;
    for (int j0 = 0; j0 < n; j0 += AHEAD) {
      uint8_t x[AHEAD][NACC];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const uint8_t* vr = cache.v + at[wave][j0 + j];
#pragma unroll
        for (int a = 0; a < NACC; ++a) x[j][a] = vr[min(lane + 64 * a, D - 1)];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float pj = ps[wave][j0 + j];
        // (rows behind the last key are the last one's: where that is NaN so is the result)
#pragma unroll
        for (int a = 0; a < NACC; ++a) acc[a] = fmaf(__builtin_amdgcn_cvt_f32_fp8((int)x[j][a], 0), pj, acc[a]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
#pragma unroll
  for (int a = 0; a < NACC; ++a)
    if (lane + 64 * a < D) sums[wave * D + lane + 64 * a] = acc[a];
  if (lane == 0) { ends[wave][0] = m; ends[wave][1] = l; }
  __syncthreads();
  float top = sink ? sink[head] : -INFINITY;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ends[w][0]);
  const float to = top == -INFINITY ? 0.f : top;
  float total = sink ? expf(sink[head] - to) : 0.f, f[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    f[w] = expf(ends[w][0] - to);
    total += ends[w][1] * f[w];
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;            // (a row without keys: zeros)
  for (int d = threadIdx.x; d < D; d += THREADS) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) a = fmaf(sums[w * D + d], f[w], a);
    out[(size_t)row * out_stride + (size_t)head * D + d] = from_float<T>(a * inv);
  }
}

extern "C" int ptl_attention_generic_f8(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k, const uint8_t* v,
                                        const float* k_scale, const float* v_scale, const int32_t* q_start, const int32_t* ctx_len,
                                        const int32_t* block_table, int bt_stride, const int32_t* work_seq, const int32_t* work_qoff,
                                        int n_work, int T, int Hq, int Hkv, int D, int page_size, int window, const float* sink,
                                        float scale, int dtype, hipStream_t stream) {
  if (n_work <= 0) return PTL_OK;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq > 65535 || D <= 0 || D > 640 || page_size <= 0 || n_work >= 1 << 26 || window < 0)
    return PTL_ERR_ARG;
  if (((uintptr_t)k | (uintptr_t)v) % (D % 16 == 0 ? 16 : D % 4 == 0 ? 4 : 1)) return PTL_ERR_ARG;
  const F8Cache cache{k, v, k_scale, v_scale};
  const F8Tables tab{q_start, ctx_len, block_table, bt_stride};
  const long groups = 16l * n_work * Hq;
  if (groups >= 1l << 31) return PTL_ERR_ARG;
  const dim3 grid((unsigned)groups);
  const bool many = (long)T * Hq > 2l * compute_units();          // (T: rows of q, a workgroup each and head)
  auto go = [&](auto kernel, int waves, auto* o, auto* x) {
    kernel<<<grid, 64 * waves, (1 + waves) * (size_t)D * sizeof(float), stream>>>(o, out_stride, x, q_stride, cache, tab, work_seq, work_qoff,
                                                                                  Hq, Hkv, D, page_size, window, sink, scale);
  };
  auto size = [&](auto* o, auto* x) {
    using T = std::remove_pointer_t<decltype(o)>;
    auto columns = [&](auto nacc) {
      constexpr int NACC = decltype(nacc)::value;
      if (many) go(attn_generic_f8_kernel<T, NACC, 4>, 4, o, x);
      else go(attn_generic_f8_kernel<T, NACC, 16>, 16, o, x);
    };
    if (D <= 64) columns(std::integral_constant<int, 1>{});
    else if (D <= 128) columns(std::integral_constant<int, 2>{});
    else if (D <= 256) columns(std::integral_constant<int, 4>{});
    else columns(std::integral_constant<int, 10>{});
  };
  if (dtype == PTL_DTYPE_F32) size((float*)out, (const float*)q);
  else if (dtype == PTL_DTYPE_BF16) size((bf16_t*)out, (const bf16_t*)q);
  else return PTL_ERR_ARG;
  return ptl_launch_status();
}

// ===========================================================================
// The matrix-core kernels: bfloat16 queries, head sizes of 32, 64, 96 and 128, pages of 16 rows and more (a power of two).
// D = 64 A + 32 B. A 16-byte piece of a key row holds, for lane group lg = lane / 16, elements 64 c + 16 lg .. +15 (c < A): the k-values of
// two matrix instructions (which k-value stands where is free, as long as the queries' agree); the last 32 elements come as
// 8 bytes, 64 A + 8 lg .. +7.

__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// two floats for another workgroup, 8-byte aligned (get_shared2 reads them)
__device__ __forceinline__ void put_shared2(float2* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, make_float2(a, b)),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// two codes (the low or the high half of x) times a power of two, as bfloat16: exact
__device__ __forceinline__ uint32_t two_bf16(uint32_t x, float scale, bool high) {
  const auto r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, scale, true)
                      : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, scale, false);
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ bf16x8_t eight_bf16(uint32_t x, uint32_t y, float scale) {
  Frag8 f;
  f.u = make_uint4(two_bf16(x, scale, false), two_bf16(x, scale, true), two_bf16(y, scale, false), two_bf16(y, scale, true));
  return f.v;
}
// the low (high) halves of two words, side by side
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// ===========================================================================
// ptl_attention_decode_f8: the sequences of a step that bring one token each.
//
// The keys of a (sequence, kv head) pair are cut into parts of ``piece`` units, the same piece for all sequences: as
// long as makes some ``cap`` parts of all of them, a workgroup a compute unit. (Sum of ceil(n_s / piece) <= cap + sequences, which
// the launch has room for.) Every workgroup finds the piece and its own part from the context lengths on the device, so a
// recorded launch suits whatever contexts it is replayed with. A pair's parts are merged by the workgroup that is done last
// (a ticket), in the order of the keys. Two parts a compute unit: 8 x 2,048 keys of 64, 8 kv heads, 10.5 us instead of 11.1, but 64 x 61 to
// 2,610 of 64 27 instead of 22, 8 x 5,000 to 7,000 of 128 31 instead of 25.
//
// A workgroup has eight waves, which take tiles of 32 keys in turn (a unit: 256), as long as there are no more pairs than the GPU runs such
// workgroups at once, two a compute unit up to D = 64, else one: what waves share in LDS need not go through memory. More pairs, then
// most of them not cut, have workgroups of four waves (a unit: 128), of which three or four run where one of eight does. us with four and
// eight: 1 x 300 of 64 5.6 5.2, 8 x 2,048 12.2 11.1, 16 x 1,000 12.9 8.6, 64 x 61 to 2,610 24.9 22.1, 128 x 300 to 1,000 21.5 22.9; 4 x 3,000
// of 128 14.2 13.4, 8 x 5,000 to 7,000 26.1 24.7, 32 x 100 to 5,000 61.7 47.4, 64 x 100 to 1,000 21.2 24.9. (Sixteen waves: 16 x 1,000 of
// 64 8.2, 8 x 2,048 11.2, 64 x 61 to 2,610 25.)
//
// What bounds it: 120,001 and 131,000 keys of 128 take 92 us, 5.6 TB/s of codes in pieces of 2 KB (a copy reaches 4.8 both ways, a
// plain stream of reads 7.1; three or four tiles a wave on their way instead of two change nothing: 2 x 120,000 89, 90, 90). Few keys: a
// chain of the context lengths, the table, the codes, and for a pair in parts of their way to memory and back, some 3 us.
//
// Both products are transposed, as in attention_decode.h:
//   S^T[key, head] = K . Q^T        A = K: lane (ln, lg) has key ln's k-values, straight from memory
//   O^T[d, head]  += V^T . P^T      B = P^T: what a lane has of S^T; A = V^T[d, key]
// A weight is rounded to bfloat16 for the second product, as over a bfloat16 cache, and the denominator sums the rounded ones (a product
// with ones), so that a row's weights add up to one: the result is off by at most 2 * 2^-8 of sum w |v|. Against 64 bits that makes an
// error of 0.0017 to 0.0022 of the result where its rounding alone makes 0.0016 to 0.0017. Weights in two parts, the rounded one and
// what it lacks, would leave that alone, with every second product twice: 64 x 61 to 2,610 of 64 22.1 23.4 us, 8 x 2,048
// 11.2 11.4, 120,001 and 131,000 of 128 92.3 93.3, a prompt of 2,048 of 64 34.8 43.1, 1,531 rows behind 6,145 keys of 128 241 366.
// Maxima, denominators and sums are float32.
// For the second a lane needs one d of the 8 keys that its P^T values belong to. It loads D / 16 neighbouring elements of each of those
// keys, which are D / 16 matrix instructions' d, and pairs the keys' halves up after the conversion (two
// v_perm_b32 for two words): no LDS between memory and the matrix cores, and nothing to wait for but the loads.
struct DecodeF8Parts {
  float *acc, *ml;                 // [part][kv head][heads of a kv head][D] sums, [..][2] their maximum and denominator
  int* tickets;                    // [sequence][kv head][head tile][TICKET]
};

constexpr int MOST_PARTS_F8 = 128; // parts of a pair
constexpr int WHOLE_F8 = 4;        // units up to which a pair is not cut: a turn is some 0.8 us, parts that meet cost 3

template <int A, int B, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, A + B <= 1 ? 4 : 3)
attn_decode_f8_kernel(const int32_t* __restrict__ ctx_len, const int32_t* __restrict__ block_table, const uint8_t* __restrict__ k_cache,
                      const uint8_t* __restrict__ v_cache, int n_seq, int Hkv, int cap, int bt_stride, int page_shift,
                      const bf16_t* __restrict__ q, long q_stride, const float* __restrict__ k_scale,
                      const float* __restrict__ v_scale, int Hq, bf16_t* __restrict__ out, long out_stride,
                      const int32_t* __restrict__ q_start, DecodeF8Parts parts, int window, const float* __restrict__ sink,
                      float scale_log2) {
  constexpr int D = 64 * A + 32 * B, NT = D / 16, STEPS = D / 32, UNIT_F8 = 32 * WAVES, THREADS = 64 * WAVES;
  constexpr int REGION = D == 32 ? 608 : 16 * D + 32;         // floats of a wave's sums
  static_assert(4 * REGION >= MOST_PARTS_F8 * 16 + 192 * 2, "the merge's weights and sums lie there too");
  __shared__ __attribute__((aligned(16))) float regions[WAVES][REGION];
  __shared__ int last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;
  const int G = Hq / Hkv, tiles = (G + 15) / 16, tile = blockIdx.y, GT = min(16, G - 16 * tile);
  const int kvh = blockIdx.x % Hkv, u = blockIdx.x / Hkv;

  // ---- which part of which sequence ----
  auto units_of = [&](int s) {
    const int c = ctx_len[s], lo = window > 0 ? max(0, c - window) : 0;
    return c > 0 ? (c - (lo & ~15) + UNIT_F8 - 1) / UNIT_F8 : 0;
  };
  int total = 0;
  for (int s0 = 0; s0 < n_seq; s0 += 64) total += s0 + lane < n_seq ? units_of(s0 + lane) : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  // (a sequence's last part is half a piece on average, so that many fewer whole ones fit ``cap`` parts)
  const int whole = max(max(cap - n_seq / 2, (3 * cap + 3) / 4), 1);
  const int piece = __builtin_amdgcn_readfirstlane(max(1, (total + whole - 1) / whole));
  int seq = -1, split = 0, n_parts = 0, before = 0;
  for (int s0 = 0; s0 < n_seq && seq < 0; s0 += 64) {
    const int units = s0 + lane < n_seq ? units_of(s0 + lane) : 0;
    const int mine = s0 + lane < n_seq ? (units <= WHOLE_F8 || !cap ? 1 : (units + piece - 1) / piece) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      upto += lane >= o ? x : 0;
    }
    const unsigned long long here = __ballot(before + upto > u);
    if (here) {
      const int at = __ffsll(here) - 1;
      seq = s0 + at;
      n_parts = __builtin_amdgcn_readlane(mine, at);
      split = u - (before + __builtin_amdgcn_readlane(upto, at) - n_parts);
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (seq < 0) return;                              // (more room than parts)
  // (the same in all lanes, which the compiler cannot see: loops, branches and addresses below become scalar)
  seq = __builtin_amdgcn_readfirstlane(seq);
  split = __builtin_amdgcn_readfirstlane(split);
  n_parts = __builtin_amdgcn_readfirstlane(n_parts);
  const int ctx = __builtin_amdgcn_readfirstlane(ctx_len[seq]), row = __builtin_amdgcn_readfirstlane(q_start[seq]);
  const int k_lo = window > 0 ? max(0, ctx - window) : 0;
  const int k_first = (k_lo & ~15) + split * piece * UNIT_F8;
  const int k_end = n_parts == 1 ? ctx : min(ctx, k_first + piece * UNIT_F8);
  const int head0 = kvh * G + 16 * tile;
  const int32_t* bt = block_table + (size_t)seq * bt_stride;
  const uint32_t page_bytes = (uint32_t)(Hkv * D) << page_shift;          // < 4 GiB, checked by the host
  const uint8_t* k_head = k_cache + ((size_t)(kvh * D) << page_shift);
  const uint8_t* v_head = v_cache + ((size_t)(kvh * D) << page_shift);

  Frag8 qf[STEPS];
  {
    const bf16_t* qr = q + (size_t)row * q_stride + (size_t)(head0 + min(ln, GT - 1)) * D;
#pragma unroll
    for (int c = 0; c < A; ++c) {
      qf[2 * c].u = load16(qr + 64 * c + 16 * lg);
      qf[2 * c + 1].u = load16(qr + 64 * c + 16 * lg + 8);
    }
    if (B) qf[2 * A].u = load16(qr + 64 * A + 8 * lg);
  }
  Frag8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones.v[j] = (__bf16)1.0f;

  struct Tile {
    uint4 k[2][A ? A : 1];
    uint2 kb[2];
    uint32_t v[2][4][A ? A : 1], vb[2][4];
    float ks[2], vs[2];
  };
  const int turns = (k_end - k_first + UNIT_F8 - 1) / UNIT_F8;          // (0: no keys)
  auto first_key = [&](int turn) { return k_first + turn * UNIT_F8 + 32 * wave; };
  // the page of the 16 keys from kp on (one page: pages hold a multiple of 16); of keys that are none, that of one that is
  auto page_at = [&](int kp) {
    const int at = __builtin_amdgcn_readfirstlane(min(max(kp, k_lo), k_end - 1) >> page_shift);
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(bt + at);
  };
  auto load = [&](Tile& t, int turn, const int (&page)[2]) __attribute__((always_inline)) {
    const int kc = first_key(turn);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int in_page = (kc + 16 * h) & ((1 << page_shift) - 1);
      const uint64_t at = (uint64_t)(uint32_t)page[h] * page_bytes + (uint32_t)(in_page * D);
      const uint8_t *kr = k_head + at, *vr = v_head + at;
      const size_t block = (size_t)page[h] * Hkv + kvh;
      t.ks[h] = *(const __attribute__((address_space(4))) float*)(uintptr_t)(k_scale + block);
      t.vs[h] = *(const __attribute__((address_space(4))) float*)(uintptr_t)(v_scale + block);
#pragma unroll
      for (int c = 0; c < A; ++c) t.k[h][c] = load_once(kr + (uint32_t)(ln * D + 64 * c + 16 * lg));
      if (B) t.kb[h] = *reinterpret_cast<const uint2*>(kr + (uint32_t)(ln * D + 64 * A + 8 * lg));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = (uint32_t)((4 * lg + i) * D);
        if constexpr (A == 1) t.v[h][i][0] = *reinterpret_cast<const uint32_t*>(vr + (x + 4 * ln));
        if constexpr (A == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(vr + (x + 8 * ln));
          t.v[h][i][0] = w.x;
          t.v[h][i][1] = w.y;
        }
        if (B) t.vb[h][i] = *reinterpret_cast<const uint16_t*>(vr + (x + 64 * A + 2 * ln));
      }
    }
  };

  f32x4_t o[NT + 1];                                // (the last one: the denominator, of ones for values)
#pragma unroll
  for (int t = 0; t <= NT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY;
  auto use = [&](Tile& t, int turn) __attribute__((always_inline)) {
    const int kc = first_key(turn);
    if (kc >= k_end) return;                        // (wave-uniform)
    const bool whole = kc >= k_lo && kc + 32 <= k_end;
    if (!whole) {
      // rows that are no keys: what lies there may be a NaN, and zero times NaN is one
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kc + 16 * h + 4 * lg + i;
          const bool in = key >= k_lo && key < k_end;
#pragma unroll
          for (int c = 0; c < A; ++c) t.v[h][i][c] = in ? t.v[h][i][c] : 0;
          if (B) t.vb[h][i] = in ? t.vb[h][i] : 0;
        }
    }
    f32x4_t st[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      st[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < A; ++c) {
        st[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16(t.k[h][c].x, t.k[h][c].y, t.ks[h]), qf[2 * c].v, st[h], 0, 0, 0);
        st[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16(t.k[h][c].z, t.k[h][c].w, t.ks[h]), qf[2 * c + 1].v, st[h], 0, 0, 0);
      }
      if (B) st[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16(t.kb[h].x, t.kb[h].y, t.ks[h]), qf[2 * A].v, st[h], 0, 0, 0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) st[h] *= scale_log2;
    if (!whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kc + 16 * h + 4 * lg + i;
          st[h][i] = key >= k_lo && key < k_end ? st[h][i] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = __builtin_elementwise_maximum(top, st[h][i]);
    top = max_with_lane_xor32(max_with_lane_xor16(top));
    // the maximum follows only when the scores pass it by 2^8: until then float32 sums and bfloat16 probabilities hold as well
    if (top > m_run + 8.0f) {
      const float keep = __builtin_amdgcn_exp2f(m_run - top);
      m_run = top;
#pragma unroll
      for (int n = 0; n <= NT; ++n) { o[n][0] *= keep; o[n][1] *= keep; o[n][2] *= keep; o[n][3] *= keep; }
    }
    const float to = m_run == -INFINITY ? 0.f : m_run;
    Frag8 p;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) p.v[4 * h + i] = (__bf16)__builtin_amdgcn_exp2f(st[h][i] - to);
    // V^T: word w of a lane's 8 keys holds two neighbouring d of each
    auto products = [&](int n, const uint32_t (&w)[8]) __attribute__((always_inline)) {
      Frag8 f;
      f.u = make_uint4(low_halves(w[0], w[1]), low_halves(w[2], w[3]), low_halves(w[4], w[5]), low_halves(w[6], w[7]));
      o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, p.v, o[n], 0, 0, 0);
      f.u = make_uint4(high_halves(w[0], w[1]), high_halves(w[2], w[3]), high_halves(w[4], w[5]), high_halves(w[6], w[7]));
      o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, p.v, o[n + 1], 0, 0, 0);
    };
#pragma unroll
    for (int c = 0; c < A; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = two_bf16(t.v[i >> 2][i & 3][c], t.vs[i >> 2], half);
        products(4 * c + 2 * half, w);
      }
    if (B) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = two_bf16(t.vb[i >> 2][i & 3], t.vs[i >> 2], false);
      products(4 * A, w);
    }
    o[NT] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, p.v, o[NT], 0, 0, 0);
  };

  if (turns > 0) {
    Tile ta, tb;
    int page[2];
    auto pages = [&](int turn) {
      const int kc = first_key(turn);
      page[0] = page_at(kc);
      page[1] = page_at(kc + 16);
    };
    pages(0);
    load(ta, 0, page);
    pages(1);
    for (int turn = 0; turn < turns; turn += 2) {
      if (turn + 1 < turns) { load(tb, turn + 1, page); pages(turn + 2); }
      use(ta, turn);
      if (turn + 1 < turns) {
        if (turn + 2 < turns) { load(ta, turn + 2, page); pages(turn + 3); }
        use(tb, turn + 1);
      }
    }
  }

  // ---- the waves' sums meet ----
  float* const region = regions[wave];
  if (ln < GT) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * lg + i;                  // row of the result tile: tile n holds d = 4 A r + n, the last ones 64 A + 2 r + n - 4 A
        region[ln * D + (n < 4 * A ? 4 * A * r + n : 64 * A + 2 * r + n - 4 * A)] = o[n][i];
      }
    if (lg == 0) { region[16 * D + 2 * ln] = m_run; region[16 * D + 2 * ln + 1] = o[NT][0]; }
  }
  __syncthreads();
  auto write = [&](int h, int d, float m, float l, float a) {
    const int head = head0 + h;
    if (sink) {
      const float s = sink[head] * 1.4426950408889634f, top = fmaxf(m, s), to = top == -INFINITY ? 0.f : top;
      const float f = __builtin_amdgcn_exp2f(m - to);
      l = l * f + __builtin_amdgcn_exp2f(s - to);
      a *= f;
    }
    out[(size_t)row * out_stride + (size_t)head * D + d] = float_to_bf16(l == 0.f ? 0.f : a / l);       // (no keys: zeros)
  };
  const size_t group = ((size_t)u * Hkv + kvh) * G + 16 * tile;             // this part's first head
  for (int i = threadIdx.x; i < GT * D; i += THREADS) {
    const int h = i / D, d = i - h * D;
    float m = -INFINITY, l = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, regions[w][16 * D + 2 * h]);
    const float to = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(regions[w][16 * D + 2 * h] - to);
      l = fmaf(regions[w][16 * D + 2 * h + 1], f, l);
      a = fmaf(regions[w][h * D + d], f, a);
    }
    if (n_parts == 1) {
      write(h, d, m, l, a);
    } else {
      put_shared(parts.acc + (group + h) * D + d, a);
      if (d == 0) { put_shared(parts.ml + (group + h) * 2, m); put_shared(parts.ml + (group + h) * 2 + 1, l); }
    }
  }
  if (n_parts == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this wave's share of the part has reached memory
  __syncthreads();
  if (threadIdx.x == 0) last = last_part(parts.tickets + (((size_t)seq * Hkv + kvh) * tiles + tile) * TICKET, n_parts);
  __syncthreads();
  if (!last || threadIdx.x >= 256) return;
  // ---- the last workgroup of the pair merges its parts ----
  // A thread takes two columns of AHEAD parts at a time; where that leaves threads, two or four groups of them share the parts.
  // What they read first is on its way while the parts' weights are made (parts that are none weigh nothing): a part
  // lies some 2 us off.
  const size_t part_heads = (size_t)Hkv * G, first = group - (size_t)split * part_heads;
  constexpr int AHEAD = 16, PAIRS_D = D / 2;
  float* const weight = regions[0];                         // [part][GT]
  float2* const sums = reinterpret_cast<float2*>(regions[0] + MOST_PARTS_F8 * 16);
  __shared__ float totals[16], tops[16];
  const int columns = GT * PAIRS_D, group_size = columns <= 64 ? 64 : columns <= 128 ? 128 : 256;
  const int side = __builtin_amdgcn_readfirstlane(threadIdx.x / group_size), in_side = threadIdx.x & (group_size - 1);
  const int sides = 256 / group_size, turns_all = (n_parts + AHEAD - 1) / AHEAD, share = (turns_all + sides - 1) / sides * AHEAD;
  const int p_begin = side * share, p_end = min(p_begin + share, turns_all * AHEAD);       // (of a last group also none)
  float2 av[AHEAD];
  auto ask = [&](int i, int p0) __attribute__((always_inline)) {
    const uint32_t column = 2 * min(i, columns - 1);
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) av[s] = get_shared2(parts.acc + (first + min(p0 + s, n_parts - 1) * part_heads) * D + column);
  };
  if (p_begin < p_end) ask(in_side, p_begin);
  for (int h = wave; h < GT; h += 4) {                      // a wave a head, a lane a part (and a second one)
    const float* ml = parts.ml + (first + h) * 2;
    float2 e[2];
    static_assert(MOST_PARTS_F8 <= 128, "two parts a lane");
#pragma unroll
    for (int x = 0; x < 2; ++x) e[x] = lane + 64 * x < n_parts ? get_shared2(ml + (lane + 64 * x) * part_heads * 2) : make_float2(-INFINITY, 0.f);
    const float m = wave_max(fmaxf(e[0].x, e[1].x)), to = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float f = __builtin_amdgcn_exp2f(e[x].x - to);
      if (lane + 64 * x < turns_all * AHEAD) weight[(lane + 64 * x) * GT + h] = f;
      l = fmaf(e[x].y, f, l);
    }
    l = wave_sum(l);
    if (lane == 0) { totals[h] = l; tops[h] = m; }
  }
  __syncthreads();
  for (int i = in_side; i - in_side < columns; i += group_size) {
    const int h = min(i / PAIRS_D, GT - 1), d = 2 * (i % PAIRS_D);
    float2 a = make_float2(0.f, 0.f);
    for (int p0 = p_begin; p0 < p_end; p0 += AHEAD) {
      if (i != in_side || p0 != p_begin) ask(i, p0);
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        const float f = weight[(p0 + s) * GT + h];
        a.x = fmaf(av[s].x, f, a.x);
        a.y = fmaf(av[s].y, f, a.y);
      }
    }
    if (sides > 1) {                                        // (then this is the only round)
      if (side) sums[threadIdx.x - group_size] = a;
      __syncthreads();
      if (side) return;
      for (int g = 0; g < sides - 1; ++g) {
        const float2 other = sums[g * group_size + in_side];
        a.x += other.x;
        a.y += other.y;
      }
    }
    if (i < columns) {
      write(h, d, tops[h], totals[h], a.x);
      write(h, d + 1, tops[h], totals[h], a.y);
    }
  }
}

static bool f8_matrix_sizes(int Hq, int Hkv, int D, int page_size) {
  return Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= 1024 && D > 0 && D % 32 == 0 && D <= 128 && page_size >= 16 &&
         (page_size & (page_size - 1)) == 0 && (long)Hkv * D * page_size < 1l << 31;
}

// cap 0: no pair is cut (then there is no workspace)
extern "C" int ptl_attention_decode_f8(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k, const uint8_t* v,
                                       const float* k_scale, const float* v_scale, const int32_t* q_start, const int32_t* ctx_len,
                                       const int32_t* block_table, int bt_stride, float* acc, float* ml, int* tickets, int cap,
                                       int n_seq, int Hq, int Hkv, int D, int page_size, int window, const float* sink, float scale,
                                       hipStream_t stream) {
  if (n_seq <= 0) return PTL_OK;
  if (!f8_matrix_sizes(Hq, Hkv, D, page_size) || cap < 0 || cap > MOST_PARTS_F8 || n_seq >= 1 << 24 || window < 0 ||
      (cap && (!acc || !ml || !tickets || (uintptr_t)ml % 8)) || ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || q_stride % 8)
    return PTL_ERR_ARG;
  const long groups = (long)(n_seq + cap) * Hkv;
  if (groups >= 1l << 31) return PTL_ERR_ARG;
  const dim3 grid((unsigned)groups, (Hq / Hkv + 15) / 16);
  int shift = 0;
  while (1 << shift < page_size) ++shift;
  const DecodeF8Parts parts{acc, ml, tickets};
  auto go = [&](auto kernel, int threads) {
    kernel<<<grid, threads, 0, stream>>>(ctx_len, block_table, k, v, n_seq, Hkv, cap, bt_stride, shift, (const bf16_t*)q, q_stride, k_scale,
                                         v_scale, Hq, (bf16_t*)out, out_stride, q_start, parts, window, sink, scale * 1.4426950408889634f);
  };
  const bool eight = (long)n_seq * Hkv * grid.y <= (long)compute_units() * (D <= 64 ? 2 : 1);
  auto size = [&](auto a, auto b) {
    constexpr int A = decltype(a)::value, B = decltype(b)::value;
    if (eight) go(attn_decode_f8_kernel<A, B, 8>, 512);
    else go(attn_decode_f8_kernel<A, B, 4>, 256);
  };
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::integral_constant<int, 1> one{};
  if (D == 32) size(none, one);
  else if (D == 64) size(one, none);
  else if (D == 96) size(one, one);
  else size(std::integral_constant<int, 2>{}, none);
  return ptl_launch_status();
}

// ===========================================================================
// ptl_attention_prefill_f8: portions of prompts. A workgroup of four waves takes 64 RT query rows of one head, 16 RT a wave, and walks the
// keys that they see in tiles of 64. A tile's codes are turned into bfloat16 (with their scales) and lie in LDS in two buffers: in the
// turn in which tile t is used, tile t + 1 is converted into the other buffer, and tile t + 2 sets out. With registers
// between memory and the conversion it sets out at the turn's end: its codes then take no registers beside the products (us
// before and behind the products, 32 heads, when this was built: 2,048 rows of 64 36.9 35.2, 2,048 behind 2,048 of 128 in 128-row blocks 158
// 145; the conversion between the two products instead of before them spills there, 353). Products, softmax, its roundings and the layout of
// LDS are those of attention_prefill.h and of the decode kernel above: S^T = K Q^T, O^T += V^T P^T, sums of the rounded weights by one
// more product with ones.
// Of a tile every wave brings 16 rows, which lie in one page: page and scales are the wave's, in scalar registers.
//
// CUT: few blocks. Their tiles, one block's behind the other's, are dealt out evenly to the workgroups that the GPU runs at once: a
// workgroup has a part of a block, blocks as a whole, and a part of one. It writes the sums of parts to the workspace as its lanes
// hold them and, its tiles done, counts them; who is last of a block's merges them. (A part costs some 8 us, ten tiles: the writes' way
// to memory, the count, and each part's way back, which is hidden behind the addition of the one before.) us, not cut and
// cut, 32 heads, rows behind keys: blocks of 64 rows 200 behind 3,000 of 128 67.7 37.4, 512 behind 8,000 of 128 178 122, 512 behind 1,024
// of 64 23.4 22.4, but 700 of 128 (11 blocks, 16 workgroups) 19.7 21.4, 1,500 behind 500 of 64 (24, 24) 34.2 42.5; of 128 rows 512 behind
// 8,000 of 128 250 109, 1,100 behind 6,000 (9, 16) 253 180, 1,531 behind 6,145 (12, 16) 279 243, 1,600 behind 6,000 (13) 272 255, 1,700 (14)
// 278 277, 2,048 behind 2,048 (16) 141 163; 1,000 behind 8,000 of 64 (8, 24) 183 114.
//
// What bounds it: 1,531 rows behind 6,145 keys, 32 heads of 128, take 242 us in blocks of 128 rows that are cut: 173 GFLOP, 715 TFLOP/s,
// 46 % of what a large product of matrices reaches. The conversion of a tile, done once for each of the blocks that read it, and the
// softmax share the vector units (the same attention over a bfloat16 cache, without the conversion and not cut: 250).
struct PrefillF8Parts {
  float2 *acc, *ml;                // [part][head][RT][2 ND][2][thread], [part][head][RT][thread]
  int* tickets;                    // [block][head][TICKET]
  int cap;
};
constexpr int NEAR_TILES = 3;      // so far from a block's beginning and end it is not cut
constexpr int WORTH_TILES = 12;    // blocks are cut where the longest becomes so many tiles shorter

template <int ND, int RT, bool CUT>
__global__ void __launch_bounds__(256, ND <= 2 ? 3 : 2)
attn_prefill_f8_kernel(bf16_t* __restrict__ out, long out_stride, const bf16_t* __restrict__ q, long q_stride, F8Cache cache, F8Tables tab,
                       const int32_t* __restrict__ work_seq, const int32_t* __restrict__ work_qoff, int n_work, int Hq, int Hkv,
                       int page_shift, int window, const float* __restrict__ sink, float scale_log2, PrefillF8Parts parts) {
  constexpr int D = 32 * ND, BN = 64, ROWS = 64 * RT;
  constexpr int PIECES = D / 8;                     // 8-element pieces of a row: 8 codes, 16 bytes of bfloat16
  // two row tiles: registers are short, so codes go to LDS without one in between, to a place of the wave's own (its 16 rows are whole
  // kilobytes, 64 lanes of 16 bytes). us with and without, 32 heads of 128, before blocks were cut: 1,531 rows behind 6,145 keys 274 284 (cut,
  // with: 241), 2,048 behind 2,048 139 145; with one row tile 332 312, 185 171.
  constexpr bool STAGED = RT == 2 && D % 64 == 0;
  __shared__ __attribute__((aligned(16))) bf16_t Ks[2][BN * D], Vs[2][BN * D];
  __shared__ __attribute__((aligned(16))) uint8_t staged[STAGED ? 4 : 1][2][STAGED ? 16 * D : 16];
  // Piece c of row r lies at c ^ swz(r), so that what 64 lanes read at once lies in different banks: of keys a piece of 16 rows (in fours,
  // beside the next piece of other fours), of values two pieces of 8 rows. A row of 128 goes over all banks: keys need 16 places
  // there, values 8 for pairs. That takes twelve more registers for addresses, which two row tiles do not have: they share
  // r & 7, and a third of LDS's cycles are conflicts (made anew for every tile addresses cost more than that, 245 us where these take
  // 242; one row tile: 1,531 rows behind 6,145 keys, 32 heads, 312 with r & 7, 300 so).
  constexpr bool WIDE = D == 128 && RT == 1;
  auto swz = [](int r) { return PIECES % 8 == 0 ? (r & 7) : ((r >> 1) & 3); };
  auto key_swz = [&](int r) { return WIDE ? r & 15 : swz(r); };
  auto value_swz = [&](int r) { return WIDE ? 2 * (r & 7) : swz(r); };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;
  // heads run along x, which the eight dies take in turn: die c gets heads c Hq / 8 .. of which a kv head's lie together
  const int head = Hq % 8 == 0 ? (blockIdx.x % 8) * (Hq / 8) + blockIdx.x / 8 : blockIdx.x;
  const int kvh = head / (Hq / Hkv), page_mask = (1 << page_shift) - 1;
  const uint32_t page_bytes = (uint32_t)(Hkv * D) << page_shift;
  const uint8_t* k_head = cache.k + ((size_t)(kvh * D) << page_shift);
  const uint8_t* v_head = cache.v + ((size_t)(kvh * D) << page_shift);
  Frag8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones.v[j] = (__bf16)1.0f;
  const float lazy = 8.0f / scale_log2;             // (raw scores: the maximum follows only where they pass it by 2^8)
  // Wave w brings rows 16 w .. +15 of a tile: 16 D bytes side by side in one page, lane l the 8 codes from 512 i + 8 l on of them
  // (addresses that differ from another one by a constant are that one and the constant: registers are short at D = 128)
  constexpr int VALUE_STORES = D == 128 ? 2 : D == 64 ? 1 : ND;      // of D = 128 and 64: every 8 rows the same piece lies in the same place
  constexpr int KEY_STORES = WIDE ? ND : VALUE_STORES;
  int key_to[KEY_STORES], value_to[VALUE_STORES];
#pragma unroll
  for (int i = 0; i < KEY_STORES; ++i) {
    const int r = (64 * i + lane) / PIECES, c = 64 * i + lane - r * PIECES;
    key_to[i] = (16 * wave + r) * D + (c ^ key_swz(r)) * 8;
    if (i < VALUE_STORES) value_to[i] = (16 * wave + r) * D + (c ^ value_swz(r)) * 8;
  }
  auto key_store_at = [&](int i) { return key_to[i % KEY_STORES] + i / KEY_STORES * 8 * D; };
  auto value_store_at = [&](int i) { return value_to[i % VALUE_STORES] + i / VALUE_STORES * 8 * D; };
  // where this lane reads: the first product takes row 16 kt + ln, piece 4 kk + lg; the second points at row
  // 32 half + 16 j + 4 lg + ln / 4, elements 16 dt + 4 (ln % 4) .. +3
  constexpr int SWAPPED = WIDE ? 16 : PIECES % 8 == 0 ? 8 : 4;       // pieces change places within so many
  int k_at[SWAPPED / 4], v_at[SWAPPED / 2];
#pragma unroll
  for (int kk = 0; kk < SWAPPED / 4; ++kk) k_at[kk] = ln * D + 8 * ((4 * kk + lg) ^ key_swz(ln));
  {
    const int r = 4 * lg + (ln >> 2);
#pragma unroll
    for (int dt = 0; dt < SWAPPED / 2; ++dt) v_at[dt] = r * D + 8 * ((2 * dt + ((ln & 3) >> 1)) ^ value_swz(r)) + 4 * (ln & 1);
  }
  auto key_at = [&](int kk) { return k_at[kk % (SWAPPED / 4)] + kk / (SWAPPED / 4) * 8 * SWAPPED; };
  auto value_at = [&](int dt) { return v_at[dt % (SWAPPED / 2)] + dt / (SWAPPED / 2) * 8 * SWAPPED; };
  const int seen_back = window > 0 ? window : 1 << 30;

  // CUT: lane i has block i, tiles first_tile .. upto - 1 of the list's; bit i of todo: this workgroup has some of them
  int first_tile = 0, upto = 0, piece = 1, my_lo = 0, my_hi = 0;
  unsigned long long todo = 0;
  if constexpr (CUT) {
    int tiles = 0;                                  // (a block without keys has one, of none; one without rows none)
    if (lane < n_work) {
      const int seq = work_seq[lane], qoff = work_qoff[lane];
      const int qlen = tab.q_start[seq + 1] - tab.q_start[seq], ctx = tab.ctx_len[seq], rows = min(ROWS, qlen - qoff);
      const int first_q = ctx - qlen + qoff, k_lo = window > 0 ? max(0, first_q - window + 1) : 0;
      if (rows > 0) tiles = max(1, (min(ctx, first_q + rows) - k_lo / BN * BN + BN - 1) / BN);
    }
    upto = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      upto += lane >= o ? x : 0;
    }
    first_tile = upto - tiles;
    const int total = __builtin_amdgcn_readlane(upto, 63), groups = gridDim.y;
    int longest = tiles;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) longest = max(longest, __shfl_xor(longest, o, 64));
    longest = __builtin_amdgcn_readfirstlane(longest);
    piece = max(NEAR_TILES + 1, (total + groups - 1) / groups);
    if (longest - piece < WORTH_TILES && n_work <= groups) {
      // a workgroup a block
      piece = my_hi = 1 << 30;
      todo = __ballot(tiles > 0 && lane == (int)blockIdx.y);
    } else {
      // where workgroup w begins: at tile w piece, or at a block's beginning or end that is near
      auto begin = [&](int w) {
        const int x = min(w * piece, total);
        const unsigned long long near = __ballot(tiles > 0 && x < total && abs(x - first_tile) <= NEAR_TILES);
        if (near) return __builtin_amdgcn_readlane(first_tile, __ffsll(near) - 1);
        return total - x <= NEAR_TILES ? total : x;
      };
      my_lo = begin(blockIdx.y);
      my_hi = begin(blockIdx.y + 1);
      todo = __ballot(tiles > 0 && first_tile < my_hi && upto > my_lo);
    }
  }
  constexpr int WORDS = RT * 2 * ND * 2 * 256, ENDS = RT * 256;                  // of a part
  unsigned long long cut_items = 0;                 // the blocks of which this workgroup has a part
  // how many parts a block has, and the workgroup of the first: workgroups begin inside of it unless near its ends
  auto parts_of = [&](int item, int& n_parts, int& first_group) {
    const int inside = (__builtin_amdgcn_readlane(first_tile, item) + NEAR_TILES + piece) / piece;
    n_parts = max(0, (__builtin_amdgcn_readlane(upto, item) - NEAR_TILES - 1) / piece - inside + 1) + 1;
    first_group = inside - 1;
  };
  // what a lane has of row tile r of a block whose rows begin at row0
  auto write = [&](int row0, int rows, int r, const f32x4_t* o, float m, float l) __attribute__((always_inline)) {
    if (sink && sink[head] > -INFINITY) l += __builtin_amdgcn_exp2f(sink[head] * 1.4426950408889634f - m * scale_log2);
    const int mine = 16 * (RT * wave + r) + ln;
    if (mine >= rows) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    bf16_t* to = out + (size_t)(row0 + mine) * out_stride + (size_t)head * D + 4 * lg;
#pragma unroll
    for (int dt = 0; dt < 2 * ND; ++dt) {
      union { uint2 u; bf16_t e[4]; } x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.e[i] = float_to_bf16(o[dt][i] * inv);
      *reinterpret_cast<uint2*>(to + 16 * dt) = x.u;
    }
  };
  // not cut: the list is sorted, most keys first; the workgroups of a head walk it forwards and backwards in turn
  for (int round = 0;; ++round) {
    const int item = CUT ? (todo ? __ffsll(todo) - 1 : n_work)
                         : round * gridDim.y + ((round & 1) ? gridDim.y - 1 - blockIdx.y : blockIdx.y);
    if (item >= n_work) break;
    todo &= todo - 1;
    const int seq = work_seq[item], qoff = work_qoff[item];
    const int first = tab.q_start[seq], qlen = tab.q_start[seq + 1] - first, ctx = tab.ctx_len[seq];
    const int rows = min(ROWS, qlen - qoff);
    if (rows <= 0) continue;
    const int32_t* bt = tab.block_table + (size_t)seq * tab.bt_stride;
    const int first_q = ctx - qlen + qoff;          // position of the block's first row
    int qpos[RT];
    Frag8 qf[RT][ND];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int mine = 16 * (RT * wave + r) + ln;
      const int qrow = mine < rows ? mine : 0;      // (rows behind the end repeat the first; they are not stored)
      qpos[r] = first_q + qrow;
      const bf16_t* x = q + (size_t)(first + qoff + qrow) * q_stride + (size_t)head * D + 8 * lg;
#pragma unroll
      for (int kk = 0; kk < ND; ++kk) qf[r][kk].u = load16(x + 32 * kk);
    }
    const int wave_first = 16 * RT * wave;
    const bool wave_has_rows = wave_first < rows;
    const int min_q = first_q + (wave_has_rows ? wave_first : 0), max_q = first_q + min(rows, wave_first + 16 * RT) - 1;
    const int wave_lo = window > 0 ? max(0, min_q - window + 1) : 0, wave_lo_last = window > 0 ? max(0, max_q - window + 1) : 0;
    f32x4_t o[RT][2 * ND + 1];
    float m_run[RT];
    const int k_lo = window > 0 ? max(0, first_q - window + 1) : 0, k_end = min(ctx, first_q + rows);
    const int k_begin = k_lo / BN * BN, n_all = max(0, (k_end - k_begin + BN - 1) / BN);
    int t_first = 0, n_tiles = n_all, n_parts = 1;   // this workgroup's tiles of the block
    if constexpr (CUT) {
      int first_group;
      parts_of(item, n_parts, first_group);
      const int begin = __builtin_amdgcn_readlane(first_tile, item);
      t_first = max(my_lo - begin, 0);
      n_tiles = min(n_all, my_hi - begin);
    }

    uint2 kc[ND], vc[ND];
    float ks, vs;
    int page;
    auto load_page = [&](int t) {
      const int kp = min(max(k_begin + t * BN + 16 * wave, k_lo), max(k_end - 1, 0));     // (of rows that are no keys: of one that is)
      page = *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(bt + __builtin_amdgcn_readfirstlane(kp >> page_shift));
    };
    auto load = [&](int t) __attribute__((always_inline)) {
      const uint64_t at = (uint64_t)(uint32_t)page * page_bytes + (uint32_t)(((k_begin + t * BN + 16 * wave) & page_mask) * D);
      const uint8_t *kr = k_head + at, *vr = v_head + at;
      if constexpr (STAGED) {
        auto to_lds = [&](const uint8_t* from, uint8_t* to) {
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (uint32_t)(16 * lane)),
                                           (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        };
#pragma unroll
        for (int i = 0; i < ND / 2; ++i) {
          to_lds(kr + 1024 * i, &staged[wave][0][1024 * i]);
          to_lds(vr + 1024 * i, &staged[wave][1][1024 * i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          kc[i] = *reinterpret_cast<const uint2*>(kr + (uint32_t)(512 * i + 8 * lane));
          vc[i] = *reinterpret_cast<const uint2*>(vr + (uint32_t)(512 * i + 8 * lane));
        }
      }
      const size_t block = (size_t)page * Hkv + kvh;
      ks = *(const __attribute__((address_space(4))) float*)(uintptr_t)(cache.k_scale + block);
      vs = *(const __attribute__((address_space(4))) float*)(uintptr_t)(cache.v_scale + block);
    };
    auto convert = [&](int t, bf16_t* Kb, bf16_t* Vb) __attribute__((always_inline)) {
      const int k0 = k_begin + t * BN + 16 * wave;
      if constexpr (STAGED) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the wave's codes have landed
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          kc[i] = *reinterpret_cast<const uint2*>(&staged[wave][0][512 * i + 8 * lane]);
          vc[i] = *reinterpret_cast<const uint2*>(&staged[wave][1][512 * i + 8 * lane]);
        }
      }
      if (k0 < k_lo || k0 + 16 > k_end) {           // rows that are no keys read as zeros (what lies there may be a NaN)
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const int k = k0 + (64 * i + lane) / PIECES;
          if (k < k_lo || k >= k_end) kc[i] = vc[i] = make_uint2(0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        *reinterpret_cast<bf16x8_t*>(Kb + key_store_at(i)) = eight_bf16(kc[i].x, kc[i].y, ks);
        *reinterpret_cast<bf16x8_t*>(Vb + value_store_at(i)) = eight_bf16(vc[i].x, vc[i].y, vs);
      }
      // what was read is in registers: the next tile's codes may come to its place (free here: the products read none of it)
      if constexpr (STAGED) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    // MASKED: some row does not see some key. CAREFUL: and a value may be a NaN
    auto tile = [&](int k0, const bf16_t* Kb, const bf16_t* Vb, auto masked_tag, auto careful_tag) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_tag)::value, CAREFUL = decltype(careful_tag)::value;
      f32x4_t st[RT][4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int r = 0; r < RT; ++r) st[r][kt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < ND; ++kk) {
          Frag8 a;
          a.u = *reinterpret_cast<const uint4*>(Kb + 16 * kt * D + key_at(kk));
#pragma unroll
          for (int r = 0; r < RT; ++r) st[r][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, qf[r][kk].v, st[r][kt], 0, 0, 0);
        }
      }
      auto transposed = [&](const bf16_t* x) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)x);
      };
      // half of the values are on their way while the softmax is made (us without and with it, rows behind keys, three runs of each within
      // 0.1: 1,024 behind 1,000 of 128 49.5 48.6, 512 behind 1,024 of 64 22.4 22.0; 2,048 of 64 35.2 35.2, 2,048 behind 3,000 of 64 110.7
      // 111.0, 2,048 of 128 65.5 65.2; keys before the conversion as well costs a quarter)
      Frag8 early[RT == 1 ? 2 * ND : 1];
      if constexpr (RT == 1 && !CAREFUL) {
#pragma unroll
        for (int dt = 0; dt < 2 * ND; ++dt) {
          early[dt].s[0] = transposed(Vb + value_at(dt));
          early[dt].s[1] = transposed(Vb + 16 * D + value_at(dt));
        }
      }
      Frag8 p[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (MASKED) {
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = k0 + 16 * kt + 4 * lg + i;
              st[r][kt][i] = k <= qpos[r] && k < k_end && k > qpos[r] - seen_back ? st[r][kt][i] : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = __builtin_elementwise_maximum(top, st[r][kt][i]);
        top = max_with_lane_xor32(max_with_lane_xor16(top));
        if (top > m_run[r] + lazy) {
          const float keep = __builtin_amdgcn_exp2f((m_run[r] - top) * scale_log2);
          m_run[r] = top;
#pragma unroll
          for (int t = 0; t <= 2 * ND; ++t) { o[r][t][0] *= keep; o[r][t][1] *= keep; o[r][t][2] *= keep; o[r][t][3] *= keep; }
        }
        const float mc = (MASKED && m_run[r] == -INFINITY) ? 0.f : -m_run[r] * scale_log2;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              p[r][half].v[4 * t + i] = (__bf16)__builtin_amdgcn_exp2f(fmaf(st[r][2 * half + t][i], scale_log2, mc));
      }
      if constexpr (CAREFUL) {
        // a NaN goes in as zero, and a product of ones for NaNs with ones for the keys that a row sees counts those it is to have
#pragma unroll
        for (int dt = 0; dt < 2 * ND; ++dt) {
          f32x4_t nans[RT];
#pragma unroll
          for (int r = 0; r < RT; ++r) nans[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            Frag8 a, is_nan;
            a.s[0] = transposed(Vb + 32 * half * D + value_at(dt));
            a.s[1] = transposed(Vb + (32 * half + 16) * D + value_at(dt));
            auto split = [](uint32_t& x) {          // codes are finite or a NaN: one if the exponent's bits are all set
              const uint32_t both = ((((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
              x &= ~both;
              return both & 0x3f803f80u;
            };
            is_nan.u = make_uint4(split(a.u.x), split(a.u.y), split(a.u.z), split(a.u.w));
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              Frag8 seen;
              int first = k0 + 32 * half + 4 * lg;
              asm("" : "+v"(first));              // (made anew for every piece of values: kept they take registers that the other products need)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int k = first + 16 * (j >> 2) + (j & 3);
                seen.v[j] = (__bf16)(k <= qpos[r] && k < k_end && k > qpos[r] - seen_back ? 1.0f : 0.0f);
              }
              o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, p[r][half].v, o[r][dt], 0, 0, 0);
              nans[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(is_nan.v, seen.v, nans[r], 0, 0, 0);
            }
          }
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][dt][i] = nans[r][i] > 0.f ? __uint_as_float(0x7fc00000u) : o[r][dt][i];
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            o[r][2 * ND] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, p[r][half].v, o[r][2 * ND], 0, 0, 0);
        return;
      }
      // (two row tiles leave no registers for values that are read early)
      if constexpr (RT == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int dt = 0; dt < 2 * ND; ++dt) {
          Frag8 a;
          if (RT == 1 && half == 0) {
            a = early[dt];
          } else {
            a.s[0] = transposed(Vb + 32 * half * D + value_at(dt));
            a.s[1] = transposed(Vb + (32 * half + 16) * D + value_at(dt));
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, p[r][half].v, o[r][dt], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) o[r][2 * ND] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones.v, p[r][half].v, o[r][2 * ND], 0, 0, 0);
      }
    };
    auto turn = [&](int t, int buffer) __attribute__((always_inline)) {
      const int k0 = k_begin + t * BN;
      if (t + 1 < n_tiles) {
        convert(t + 1, Ks[1 - buffer], Vs[1 - buffer]);
        if constexpr (STAGED) {
          if (t + 2 < n_tiles) { load(t + 2); load_page(t + 3); }
        }
      }
      if (wave_has_rows && k0 <= max_q && k0 + BN > wave_lo) {
        const bool need_mask = k0 + BN - 1 > min_q || k0 + BN > k_end || k0 < wave_lo_last;
        if (need_mask) tile(k0, Ks[buffer], Vs[buffer], std::true_type{}, std::false_type{});
        else tile(k0, Ks[buffer], Vs[buffer], std::false_type{}, std::false_type{});
      }
      if (!STAGED && t + 2 < n_tiles) { load(t + 2); load_page(t + 3); }
      __syncthreads();
    };
    auto begin_sums = [&] {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        m_run[r] = -INFINITY;
#pragma unroll
        for (int t = 0; t <= 2 * ND; ++t) o[r][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
    };
    begin_sums();
    if (t_first < n_tiles) {
      load_page(t_first);
      load(t_first);
      load_page(t_first + 1);
      convert(t_first, Ks[0], Vs[0]);
      if (t_first + 1 < n_tiles) { load(t_first + 1); load_page(t_first + 2); }
    }
    __syncthreads();
    for (int t = t_first; t < n_tiles; t += 2) {
      turn(t, 0);
      if (t + 1 < n_tiles) turn(t + 1, 1);
    }
    // A value that is a NaN makes one of every row that its tile's products go to, also of rows that do not see its key: zero times
    // NaN is one. Where sums are NaNs the block is taken again with the careful products (by the workgroup's waves
    // together); where they are not, all that costs is to look at them once a block (us without and with it, 32 heads: 2,048 rows of 64
    // 34.9 35.2, of 128 64.9 65.2, 1,531 behind 6,145 keys of 128 242.6 243.2; 1,024 behind 4,000 of 64, blocks of 128 rows whose registers
    // are all taken, 72.8 75.0).
    {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < 2 * ND; ++t) sum += (o[r][t][0] + o[r][t][1]) + (o[r][t][2] + o[r][t][3]);
      // (the second buffer: its last reader has passed the last turn's barrier, its next writer comes behind another one)
      int* const found = reinterpret_cast<int*>(Ks[1]);
      const bool here = __any(sum != sum);
      if (lane == 0) found[wave] = here;
      __syncthreads();
      if (__builtin_amdgcn_readfirstlane(found[0] | found[1] | found[2] | found[3])) {
        begin_sums();
        for (int t = t_first; t < n_tiles; ++t) {
          const int k0 = k_begin + t * BN;
          load_page(t);
          load(t);
          convert(t, Ks[0], Vs[0]);
          __syncthreads();
          if (wave_has_rows && k0 <= max_q && k0 + BN > wave_lo) tile(k0, Ks[0], Vs[0], std::true_type{}, std::true_type{});
          __syncthreads();
        }
      }
    }
    if constexpr (CUT) {
      if (n_parts > 1) {
        cut_items |= 1ull << item;
        const size_t mine = (size_t)(blockIdx.y + item) * Hq + head;         // (workgroup + block: goes up from part to part)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
          for (int dt = 0; dt < 2 * ND; ++dt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              put_shared2(parts.acc + mine * WORDS + ((r * 2 * ND + dt) * 2 + x) * 256 + threadIdx.x, o[r][dt][2 * x], o[r][dt][2 * x + 1]);
          put_shared2(parts.ml + mine * ENDS + r * 256 + threadIdx.x, m_run[r], o[r][2 * ND][0]);
        }
        continue;
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) write(first + qoff, rows, r, o[r], m_run[r], o[r][2 * ND][0]);
  }
  if constexpr (CUT) {
    // ---- parts: at most two, the end of a block and the beginning of one ----
    if (!cut_items) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this wave's share of them has reached memory
    __syncthreads();
    int* const told = reinterpret_cast<int*>(Ks[0]);          // (LDS is full to the last byte, and nobody reads keys any more)
    int* ticket = nullptr;
    int of = 0;
    unsigned long long left = cut_items;
    for (int i = 0; left; ++i, left &= left - 1) {
      const int item = __ffsll(left) - 1;
      int n_parts, first_group;
      parts_of(item, n_parts, first_group);
      if ((int)threadIdx.x == i) {
        ticket = parts.tickets + ((size_t)item * Hq + head) * TICKET;
        of = n_parts;
      }
    }
    if (ticket) told[threadIdx.x] = last_part(ticket, of);
    __syncthreads();
    for (int i = 0; cut_items; ++i, cut_items &= cut_items - 1) {
      if (!__builtin_amdgcn_readfirstlane(told[i])) continue;
      const int item = __ffsll(cut_items) - 1;
      int n_parts, first_group;
      parts_of(item, n_parts, first_group);
      const int seq = work_seq[item], qoff = work_qoff[item], first = tab.q_start[seq], rows = min(ROWS, tab.q_start[seq + 1] - first - qoff);
      const size_t first_part = (size_t)(first_group + item) * Hq + head;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        // in the order of the keys; while one part is added the next one is on its way
        struct Part { float2 ml, acc[4 * ND]; };
        Part even, odd;
        auto bring = [&](Part& x, int p) __attribute__((always_inline)) {
          const size_t at = first_part + (size_t)p * Hq;
          x.ml = get_shared2((const float*)(parts.ml + at * ENDS + r * 256 + threadIdx.x));
#pragma unroll
          for (int j = 0; j < 4 * ND; ++j) x.acc[j] = get_shared2((const float*)(parts.acc + at * WORDS + (r * 4 * ND + j) * 256 + threadIdx.x));
        };
        f32x4_t o[2 * ND];
#pragma unroll
        for (int dt = 0; dt < 2 * ND; ++dt) o[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        auto add = [&](const Part& x) __attribute__((always_inline)) {
          // (a part that has seen no key has zero sums and a maximum of -inf)
          const float top = max2(m, x.ml.x), to = top == -INFINITY ? 0.f : top;
          const float keep = __builtin_amdgcn_exp2f((m - to) * scale_log2), f = __builtin_amdgcn_exp2f((x.ml.x - to) * scale_log2);
          m = top;
          l = fmaf(l, keep, x.ml.y * f);
#pragma unroll
          for (int dt = 0; dt < 2 * ND; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[dt][j] = fmaf(o[dt][j], keep, (j & 1 ? x.acc[2 * dt + j / 2].y : x.acc[2 * dt + j / 2].x) * f);
        };
        bring(even, 0);
        for (int p = 0; p < n_parts; p += 2) {
          if (p + 1 < n_parts) bring(odd, p + 1);
          add(even);
          if (p + 1 < n_parts) {
            if (p + 2 < n_parts) bring(even, p + 2);
            add(odd);
          }
        }
        write(first + qoff, rows, r, o, m, l);
      }
    }
  }
}

// cap > 0: blocks are cut into some ``cap`` parts a head in all (n_work up to 64; work: (n_work + cap) * Hq * block_rows *
// (D + 8) floats, tickets: n_work * Hq * TICKET zeros, zeros again afterwards). Else ``groups`` workgroups a head take whole blocks.
extern "C" int ptl_attention_prefill_f8(void* out, long out_stride, const void* q, long q_stride, const uint8_t* k, const uint8_t* v,
                                        const float* k_scale, const float* v_scale, const int32_t* q_start, const int32_t* ctx_len,
                                        const int32_t* block_table, int bt_stride, const int32_t* work_seq, const int32_t* work_qoff,
                                        int n_work, int groups, int cap, float* work, int* tickets, int block_rows, int Hq, int Hkv,
                                        int D, int page_size, int window, const float* sink, float scale, hipStream_t stream) {
  if (n_work <= 0) return PTL_OK;
  if (!f8_matrix_sizes(Hq, Hkv, D, page_size) || window < 0 || groups <= 0 || groups > 65535 || (block_rows != 64 && block_rows != 128) ||
      !(scale > 0.f) || ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || q_stride % 8 || (uintptr_t)out % 8 || out_stride % 4)
    return PTL_ERR_ARG;
  if (cap < 0 || (cap && (n_work > 64 || cap > 4096 || !work || (uintptr_t)work % 8 || !tickets))) return PTL_ERR_ARG;
  const F8Cache cache{k, v, k_scale, v_scale};
  const F8Tables tab{q_start, ctx_len, block_table, bt_stride};
  const PrefillF8Parts parts{(float2*)work, (float2*)(work + (size_t)(n_work + cap) * Hq * block_rows * D), tickets, cap};
  int shift = 0;
  while (1 << shift < page_size) ++shift;
  auto go = [&](auto kernel, int y) {
    kernel<<<dim3(Hq, y), 256, 0, stream>>>((bf16_t*)out, out_stride, (const bf16_t*)q, q_stride, cache, tab, work_seq, work_qoff, n_work,
                                            Hq, Hkv, shift, window, sink, scale * 1.4426950408889634f, parts);
  };
  auto size = [&](auto nd) {
    constexpr int ND = decltype(nd)::value;
    if (block_rows == 64) {
      if (cap) go(attn_prefill_f8_kernel<ND, 1, true>, cap);
      else go(attn_prefill_f8_kernel<ND, 1, false>, groups);
    } else {
      if (cap) go(attn_prefill_f8_kernel<ND, 2, true>, cap);
      else go(attn_prefill_f8_kernel<ND, 2, false>, groups);
    }
  };
  if (D == 32) size(std::integral_constant<int, 1>{});
  else if (D == 64) size(std::integral_constant<int, 2>{});
  else if (D == 96) size(std::integral_constant<int, 3>{});
  else size(std::integral_constant<int, 4>{});
  return ptl_launch_status();
}
