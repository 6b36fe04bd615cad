// Pages of a cache: the store of a step's keys and values into pages held in 8 bits, and copies of pages.
//
// A block is what a page holds of one kv head, page_size rows of D; keys and values have blocks, and scales, of their own.
// A block stands for the numbers e4m3(code) * scale, scale = 2^e the smallest power of two, e >= -126, with |x| <= 448 scale
// for every finite x that was stored into it. (A number of e4m3's normal range, |x| >= 2^-6 scale, is then rounded to four
// significant bits whatever the scale is: what the other tokens of a block change of it lies below 2^-14 of the block's
// largest number. With a scale of largest / 448 all numbers of a block would move with its largest.) What is not finite is
// stored as NaN and takes no part in the scale.
#include "common.h"
#include "device.h"
#include <type_traits>

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The exponent of the scale of numbers up to ``largest`` (finite, not negative): 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float largest) {
  const uint32_t u = __float_as_uint(largest);
  return max(-126, (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// two numbers as e4m3 codes in the low 16 bits: |x| <= 448, or not finite (then NaN). Rounds to nearest even.
__device__ __forceinline__ uint32_t two_codes(float a, float b) {
  a = fabsf(a) <= 448.f ? a : __uint_as_float(0x7fc00000u);
  b = fabsf(b) <= 448.f ? b : __uint_as_float(0x7fc00000u);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// ===========================================================================
// ptl_rope_store_f8: the rotation of csrc/rope.hip (same angles, same formula), the queries rounded to their type, the keys and
// the values into their blocks.
//
// The tokens of a page that a call brings are a run: rows one after the other with slots one after the other. A run that
// begins at its page's first row begins the block anew (the old scale counts no more and the rows behind the run become
// zeros); one that begins further back takes the block as it is, and where the new tokens need a larger scale the other rows'
// codes are rounded anew to it. So a block's content does not depend on how often the same run is stored.
//
// The first workgroups store, a wave a task (row that begins a run, kv head, keys or values): a block belongs to one wave and no two
// waves write one scale. Up to DIRECT rows every row has its tasks, and the waves of rows that begin nothing leave. Beyond, a
// workgroup makes the list of the rows that begin a run (of LISTED rows at a time) and its waves take their share of the
// tasks; with a workgroup for every row 2,048 rows, 8 kv heads of 128, took 71 us, from lists they took 17.6, and where the four tasks of a
// workgroup are of one run, whose angles they make together, they take 15.0.
// A wave takes the rows of its run a chunk at a time, holds their numbers of a head and finds the largest; a run of one chunk (16 rows
// of 128) is then written from the registers, a longer one read and rotated again. Behind them the workgroups that rotate the queries, a
// row a wave.
constexpr int DIRECT = 128;
constexpr int LISTED = 2048;
constexpr int ANGLES = 1024;         // cosines and sines that a wave keeps in LDS, and pairs that it holds: the rows of a chunk

// The factor that row m of q, k and v still lacks (ops.RowScale): rsqrt(sum_j partials[m][j] / size + eps); partials == null: none. For the
// few rows of a decode step, whose norm is finished by who reads its product.
constexpr int SCALED_ROWS = 16;      // no more than DIRECT
struct RowFactor {
  const float* partials;           // [T, count]
  int count;
  float inv_size, eps;
  // by a whole wave
  __device__ __forceinline__ float of(int m, int lane) const {
    float sum = 0.f;
    for (int j = lane; j < count; j += 64) sum += partials[(size_t)m * count + j];
    return rsqrtf(wave_sum(sum) * inv_size + eps);
  }
};

// The run that begins at row t0, if one does: its keys or values of head h. A wave's work, or (TEAM) that of the workgroup's four. SHARED: the
// workgroup's waves are at the same run, of one chunk, and make its angles together.
template <typename T, int VEC, bool TEAM, bool SHARED, bool SCALED>
__device__ __forceinline__ void
store_run(int t0, int h, bool values, int lane, int wave, float2* __restrict__ table, float* __restrict__ largest_of_wave, const T* __restrict__ k, const T* __restrict__ v,
          long row_stride, const int32_t* __restrict__ positions, const float* __restrict__ inv_freq,
          const int32_t* __restrict__ slots, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
          float* __restrict__ k_scale, float* __restrict__ v_scale, int T_, int Hkv, int D, int page_size, int slots_in_all,
          const RowFactor& factor, float* __restrict__ row_factor) {
  struct __attribute__((aligned(sizeof(T) * VEC))) Vec { T e[VEC]; };
  constexpr int HELD = ANGLES / 64 / VEC;                        // items of VEC pairs a lane has of a chunk
  constexpr int WAVES = TEAM ? 4 : 1;
  const int w = TEAM ? wave : 0;
  const int half = D >> 1, per_row = half / VEC, chunk = ANGLES / half;       // items in a row of D, rows of a chunk
  const T* from = (values ? v : k) + (size_t)t0 * row_stride + h * D;
  const bool turn = inv_freq && !values;
  // the slots from the row before on, a lane each
  const int near = t0 - 1 + lane;
  const int seen = near >= 0 && near < T_ ? slots[near] : -2;
  const int slot = __builtin_amdgcn_readlane(seen, 1), before = __builtin_amdgcn_readlane(seen, 0);
  const int page = slot / page_size, off = slot - page * page_size;
  if (slot < 0 || slot >= slots_in_all || (before >= 0 && before == slot - 1 && off > 0)) return;     // no run begins here
  const int most = min(page_size - off, T_ - t0);
  int n;                                                         // rows of the run
  {
    const unsigned long long stop = ~(__ballot(lane <= most && seen == slot + lane - 1) | 1ull);      // (the first row without a next slot)
    n = stop ? __ffsll(stop) - 2 : 63;
    for (; n >= 63 && n < most; n += 64) {
      const bool next = n + lane < most && slots[t0 + n + lane] == slot + n + lane;
      const unsigned long long end = ~__ballot(next);
      if (end) { n += __ffsll(end) - 1; break; }
    }
    n = __builtin_amdgcn_readfirstlane(min(n, most));
  }
  float* scale = (values ? v_scale : k_scale) + (size_t)page * Hkv + h;
  uint8_t* const rows = (values ? v_cache : k_cache) + ((size_t)page * Hkv + h) * page_size * D;
  const float old = off > 0 ? *scale : 0.f;

  auto meet = [] {
    if constexpr (SHARED) {
      __syncthreads();
    } else {                                                      // (a wave's own LDS)
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  };
  // rows r0 .. of the run, as many as a chunk has: a and b hold item lane + 64 it of them, VEC pairs of one row
  auto load = [&](int r0, float (&a)[HELD][VEC], float (&b)[HELD][VEC]) __attribute__((always_inline)) {
    const int count = min(chunk, n - r0), items = count * per_row;
    Vec x[HELD], y[HELD];
#pragma unroll
    for (int it = 0; it < HELD; ++it) {
      const int i = min(lane + 64 * it, items - 1), r = i / per_row;
      const T* at = from + (size_t)(r0 + r) * row_stride + (i - r * per_row) * VEC;
      x[it] = *reinterpret_cast<const Vec*>(at);
      y[it] = *reinterpret_cast<const Vec*>(at + half);
    }
    if constexpr (SCALED) {
      for (int r = 0; r < count; ++r) {
        const float f = factor.of(t0 + r0 + r, lane);
        if (lane == 0) row_factor[r] = f;
      }
    }
    if (SHARED ? inv_freq != nullptr : turn) {
      // the angles' cosines and sines once for the chunk, an angle a lane (sincosf is some hundred instructions: in the loop below
      // they would be 16 times as many, and a launch that has one row a wave is the time of fetching them)
      for (int i = SHARED ? threadIdx.x : lane; i < count * half; i += SHARED ? 256 : 64) {
        const int r = i / half;
        float s, c;
        sincosf((float)positions[t0 + r0 + r] * inv_freq[i - r * half], &s, &c);
        table[i] = make_float2(c, s);
      }
    }
    meet();                                                       // (LDS: written above, read below)
#pragma unroll
    for (int it = 0; it < HELD; ++it) {
      const int i = min(lane + 64 * it, items - 1);
      float f = 1.f;
      if constexpr (SCALED) f = row_factor[i / per_row];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float x1 = to_float<T>(x[it].e[e]), x2 = to_float<T>(y[it].e[e]);
        if constexpr (SCALED) { x1 *= f; x2 *= f; }
        float2 cs = make_float2(1.f, 0.f);
        if (turn) cs = table[i * VEC + e];                        // (row r's pairs begin at r * half)
        a[it][e] = turn ? x1 * cs.x - x2 * cs.y : x1;
        b[it][e] = turn ? x2 * cs.x + x1 * cs.y : x2;
      }
    }
    meet();
    return items;
  };
  auto largest_of = [&](const float (&a)[VEC], float m) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x = fabsf(a[e]);
      m = x < INFINITY ? fmaxf(m, x) : m;
    }
    return m;
  };
  float a[HELD][VEC], b[HELD][VEC], m = 0.f;
  int items = 0;
  for (int r0 = w * chunk; r0 < n; r0 += WAVES * chunk) {
    items = load(r0, a, b);                                       // (lanes behind the last item hold it once more)
#pragma unroll
    for (int it = 0; it < HELD; ++it) m = largest_of(b[it], largest_of(a[it], m));
  }
  m = wave_max(m);
  if constexpr (TEAM) {
    if (lane == 0) largest_of_wave[wave] = m;
    __syncthreads();                                              // (and every wave has read the scale there was)
    m = fmaxf(fmaxf(largest_of_wave[0], largest_of_wave[1]), fmaxf(largest_of_wave[2], largest_of_wave[3]));
  }
  int e_new = scale_exponent(m);
  if (off > 0) {
    const int e_old = max(-126, (int)(__float_as_uint(old) >> 23) - 127);
    if (e_old >= e_new) {
      e_new = e_old;
    } else {
      // the block's other rows are rounded anew to the larger scale (of numbers below 2^-126 of it nothing is left)
      const float f = e_old - e_new < -126 ? 0.f : power_of_two(e_old - e_new);
      auto again = [&](uint32_t x) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
        return two_codes(lo[0] * f, lo[1] * f) | two_codes(hi[0] * f, hi[1] * f) << 16;
      };
      // (the run's own rows are left to the writes below: lanes of a wave would write them in no certain order)
      auto other = [&](int i) { const int r = i / D; return r < off || r >= off + n; };
      if (D % 4 == 0) {
        for (int i = 4 * (64 * w + lane); i < page_size * D; i += 256 * WAVES)
          if (other(i)) *reinterpret_cast<uint32_t*>(rows + i) = again(*reinterpret_cast<const uint32_t*>(rows + i));
      } else {                                    // D is even: two neighbours lie in one row
        for (int i = 2 * (64 * w + lane); i < page_size * D; i += 128 * WAVES)
          if (other(i)) *reinterpret_cast<uint16_t*>(rows + i) = (uint16_t)again(*reinterpret_cast<const uint16_t*>(rows + i));
      }
    }
  } else {
    for (int i = n * D + 2 * (64 * w + lane); i < page_size * D; i += 128 * WAVES) *reinterpret_cast<uint16_t*>(rows + i) = 0;
  }
  if (w == 0 && lane == 0) *scale = power_of_two(e_new);
  const float f = power_of_two(-e_new);
  auto put = [&](int r, int j, const float (&x)[VEC], const float (&y)[VEC]) __attribute__((always_inline)) {
    uint8_t* const to = rows + (off + r) * D + j;
    if constexpr (VEC == 8) {
      uint2 lo, hi;
      lo.x = two_codes(x[0] * f, x[1] * f) | two_codes(x[2] * f, x[3] * f) << 16;
      lo.y = two_codes(x[4] * f, x[5] * f) | two_codes(x[6] * f, x[7] * f) << 16;
      hi.x = two_codes(y[0] * f, y[1] * f) | two_codes(y[2] * f, y[3] * f) << 16;
      hi.y = two_codes(y[4] * f, y[5] * f) | two_codes(y[6] * f, y[7] * f) << 16;
      *reinterpret_cast<uint2*>(to) = lo;
      *reinterpret_cast<uint2*>(to + half) = hi;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t z = two_codes(x[e] * f, y[e] * f);
        to[e] = (uint8_t)z;
        to[half + e] = (uint8_t)(z >> 8);
      }
    }
  };
  for (int r0 = w * chunk; r0 < n; r0 += WAVES * chunk) {
    if (n > WAVES * chunk) items = load(r0, a, b);
#pragma unroll
    for (int it = 0; it < HELD; ++it) {
      const int i = lane + 64 * it, r = i / per_row;
      if (i < items) put(r0 + r, (i - r * per_row) * VEC, a[it], b[it]);
    }
  }
}

template <typename T, int VEC, bool SCALED>
__global__ void __launch_bounds__(256, VEC == 8 ? 4 : 2)
rope_store_f8_kernel(T* __restrict__ q_out, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                     long row_stride, const int32_t* __restrict__ positions, const float* __restrict__ inv_freq,
                     const int32_t* __restrict__ slots, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
                     float* __restrict__ k_scale, float* __restrict__ v_scale, int T_, int Hq, int Hkv, int D, int page_size,
                     int slots_in_all, int store_groups, RowFactor factor) {
  __shared__ __attribute__((aligned(16))) float2 tables[4][ANGLES];
  __shared__ float largest_of_wave[4], row_factors[4][SCALED_ROWS];
  struct __attribute__((aligned(sizeof(T) * VEC))) Vec { T e[VEC]; };
  const int half = D >> 1, per_row = half / VEC;               // items of VEC pairs in a row of D
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= store_groups) {
    // ---- queries: a wave a row, of few rows a workgroup ----
    const int share = T_ <= DIRECT ? 4 : 1, block = blockIdx.x - store_groups;
    const int t = share == 4 ? block : 4 * block + wave;
    if (t >= T_) return;
    const T* row = q + (size_t)t * row_stride;
    T* to = q_out + (size_t)t * Hq * D;
    const int total = Hq * per_row;
    constexpr int AHEAD = VEC == 8 ? 4 : 8;
    float2* const table = tables[wave];
    float f = 1.f;
    for (int i0 = share == 4 ? 64 * wave : 0, at = i0; i0 < total; i0 += 64 * AHEAD * share) {
      Vec x[AHEAD], y[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int i = min(i0 + 64 * share * n + lane, total - 1), h = i / per_row, j = (i - h * per_row) * VEC;
        x[n] = *reinterpret_cast<const Vec*>(row + h * D + j);
        y[n] = *reinterpret_cast<const Vec*>(row + h * D + j + half);
      }
      if (SCALED && i0 == at) f = factor.of(t, lane);
      if (inv_freq && i0 == at) {                   // (the first time)
        const float pos = (float)positions[t];
        for (int j = lane; j < half; j += 64) {
          float s, c;
          sincosf(pos * inv_freq[j], &s, &c);
          table[j] = make_float2(c, s);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int i = i0 + 64 * share * n + lane;
        if (i >= total) continue;
        const int h = i / per_row, j = (i - h * per_row) * VEC;
        if (inv_freq || SCALED) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float x1 = to_float<T>(x[n].e[e]), x2 = to_float<T>(y[n].e[e]);
            if constexpr (SCALED) { x1 *= f; x2 *= f; }
            const float2 cs = inv_freq ? table[j + e] : make_float2(1.f, 0.f);
            x[n].e[e] = from_float<T>(x1 * cs.x - x2 * cs.y);
            y[n].e[e] = from_float<T>(x2 * cs.x + x1 * cs.y);
          }
        }
        *reinterpret_cast<Vec*>(to + h * D + j) = x[n];
        *reinterpret_cast<Vec*>(to + h * D + j + half) = y[n];
      }
    }
    return;
  }
  // ---- keys and values ----
  if (T_ <= DIRECT) {
    const int task = blockIdx.x * 4 + wave, t = task / (2 * Hkv), rest = task - t * 2 * Hkv;
    if (t < T_)
      store_run<T, VEC, false, false, SCALED>(t, rest >> 1, rest & 1, lane, wave, tables[wave], nullptr, k, v, row_stride, positions, inv_freq, slots,
                               k_cache, v_cache, k_scale, v_scale, T_, Hkv, D, page_size, slots_in_all, factor, row_factors[wave]);
    return;
  }
  if constexpr (!SCALED) {                         // (few rows: never here)
    __shared__ int16_t list[LISTED];
    __shared__ int counts[LISTED / 64];
    // pages of more rows than a chunk has: a workgroup a task (us, pages of 64 rows of 128, 2,048 rows: a wave a task 49.5,
    // so 16.9)
    const bool team = page_size * half > ANGLES;
    const int step = team ? store_groups : 4 * store_groups;
    int next = team ? blockIdx.x : blockIdx.x * 4 + wave;         // the next task, counted from the segment's first
    for (int seg = 0; seg < T_; seg += LISTED) {
      constexpr int TURNS = LISTED / 256;             // row seg + 256 j + threadIdx.x in turn j: all are asked for at once
      int at[TURNS], before[TURNS];
#pragma unroll
      for (int j = 0; j < TURNS; ++j) {
        const int t = seg + 256 * j + threadIdx.x;
        at[j] = t < T_ ? slots[t] : -1;
        before[j] = t > 0 && t < T_ ? slots[t - 1] : -2;
      }
      unsigned long long all[TURNS];                  // the wave's rows that begin a run
#pragma unroll
      for (int j = 0; j < TURNS; ++j) {
        all[j] = 0;
        if (seg + 256 * j < T_)
          all[j] = __ballot(at[j] >= 0 && at[j] < slots_in_all && (before[j] != at[j] - 1 || before[j] < 0 || at[j] % page_size == 0));
        if (lane == 0) counts[4 * j + wave] = __popcll(all[j]);
      }
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int j = 0; j < TURNS; ++j) {
        int first = total;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          first += w < wave ? counts[4 * j + w] : 0;
          total += counts[4 * j + w];
        }
        if (all[j] >> lane & 1) list[first + __popcll(all[j] & ((1ull << lane) - 1))] = (int16_t)(256 * j + threadIdx.x);
      }
      __syncthreads();
      total = __builtin_amdgcn_readfirstlane(total) * 2 * Hkv;
      for (; next < total; next += step) {
        const int run = next / (2 * Hkv), task = next - run * 2 * Hkv, t0 = seg + __builtin_amdgcn_readfirstlane((int)list[run]);
        auto store = [&](auto together, auto same_run, float2* table) __attribute__((always_inline)) {
          store_run<T, VEC, decltype(together)::value, decltype(same_run)::value, SCALED>(
              t0, task >> 1, task & 1, lane, wave, table, largest_of_wave, k, v, row_stride, positions, inv_freq, slots, k_cache, v_cache,
              k_scale, v_scale, T_, Hkv, D, page_size, slots_in_all, factor, row_factors[wave]);
        };
        if (team) {
          store(std::true_type{}, std::false_type{}, tables[wave]);
          __syncthreads();                            // (the waves' largest numbers have been read)
        } else if (Hkv % 2 == 0) {                    // four tasks, of one run
          store(std::false_type{}, std::true_type{}, tables[0]);
        } else {
          store(std::false_type{}, std::false_type{}, tables[wave]);
        }
      }
      next -= total;
      __syncthreads();
    }
  }
}

extern "C" int ptl_rope_store_f8(void* q_out, const void* q, const void* k, const void* v, long row_stride,
                                 const int32_t* positions, const float* inv_freq, const int32_t* slots, uint8_t* k_cache,
                                 uint8_t* v_cache, float* k_scale, float* v_scale, int T, int Hq, int Hkv, int D, int page_size,
                                 int pages, const float* partials, int count, int size, float eps, int dtype, hipStream_t stream) {
  if (T <= 0) return PTL_OK;
  if (Hq <= 0 || Hkv <= 0 || D <= 0 || (D & 1) || D > 640 || page_size <= 0 || (long)page_size * D >= 1l << 30) return PTL_ERR_ARG;
  if (slots && (!k_cache || !v_cache || !k_scale || !v_scale)) return PTL_ERR_ARG;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) % (D % 16 == 0 ? 16 : D % 4 == 0 ? 4 : 2)) return PTL_ERR_ARG;
  if (partials && (T > SCALED_ROWS || count <= 0 || size <= 0)) return PTL_ERR_ARG;
  const RowFactor factor{partials, count, partials ? 1.0f / (float)size : 0.f, eps};
  const int in_all = slots ? (int)min((long)pages * page_size, 0x7fffffffl) : 0;
  if (T >= 1 << 30 || Hkv >= 1 << 16) return PTL_ERR_ARG;
  // a wave for every task there can be, up to eight a compute unit
  const long tasks = ((long)T * 2 * Hkv + 3) / 4;
  const int store_groups = !slots ? 0 : T <= DIRECT ? (int)tasks : (int)min(tasks, 2l * compute_units());
  const int groups = (T <= DIRECT ? T : (T + 3) / 4) + store_groups;
  const bool vec = (D / 2) % 8 == 0 && row_stride % 8 == 0 && ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out) % 16 == 0;
  if (dtype == PTL_DTYPE_F32) {
    auto go = [&](auto kernel) {
      kernel<<<groups, 256, 0, stream>>>((float*)q_out, (const float*)q, (const float*)k, (const float*)v, row_stride, positions,
                                           inv_freq, slots, k_cache, v_cache, k_scale, v_scale, T, Hq, Hkv, D, page_size, in_all, store_groups, factor);
    };
    if (partials) { if (vec) go(rope_store_f8_kernel<float, 8, true>); else go(rope_store_f8_kernel<float, 1, true>); }
    else if (vec) go(rope_store_f8_kernel<float, 8, false>); else go(rope_store_f8_kernel<float, 1, false>);
  } else if (dtype == PTL_DTYPE_BF16) {
    auto go = [&](auto kernel) {
      kernel<<<groups, 256, 0, stream>>>((bf16_t*)q_out, (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, row_stride, positions,
                                           inv_freq, slots, k_cache, v_cache, k_scale, v_scale, T, Hq, Hkv, D, page_size, in_all, store_groups, factor);
    };
    if (partials) { if (vec) go(rope_store_f8_kernel<bf16_t, 8, true>); else go(rope_store_f8_kernel<bf16_t, 1, true>); }
    else if (vec) go(rope_store_f8_kernel<bf16_t, 8, false>); else go(rope_store_f8_kernel<bf16_t, 1, false>);
  } else {
    return PTL_ERR_ARG;
  }
  return ptl_launch_status();
}

// ===========================================================================
// ptl_copy_pages: page src[i] -> page dst[i] of several pools [layers, pages, page bytes], all layers, one launch. The host has
// checked that no page is written twice, or read and written. The page numbers travel with the launch (PAIRS of them; more are
// more launches), so nothing is uploaded and a recorded launch keeps its own. Memory bounds it: 64 pages of 32 KB in 32 layers, keys and
// values, 268 MB in all, 46 us (5.8 TB/s, part of it the last-level cache's); one page of 16 layers 2.7 us, a launch.
constexpr int PAIRS = 256, POOLS = 16;
struct CopyPool {
  char* at;
  long page_bytes, layer_bytes;
  uint32_t units;                  // pieces of a thread's 16, 4 or one byte in a page
  uint32_t pieces;                 // layers * pairs * units
  uint32_t first_group;            // the launch's workgroups from here on are this pool's
  uint32_t size;                   // bytes of a piece: as many as the pool's address and pages allow
};
struct CopyPages {
  CopyPool pools[POOLS];
  int n_pools, n_pairs;
  int32_t src[PAIRS], dst[PAIRS];
};

constexpr int COPY_AHEAD = 4;      // pieces that a thread asks for at once

template <typename V>
__device__ __forceinline__ void copy_pieces(const CopyPages& c, const CopyPool& pool) {
  const uint32_t first = (blockIdx.x - pool.first_group) * (256 * COPY_AHEAD) + threadIdx.x;
  V held[COPY_AHEAD];
  char* to[COPY_AHEAD];
#pragma unroll
  for (int i = 0; i < COPY_AHEAD; ++i) {
    const uint32_t piece = min(first + 256 * i, pool.pieces - 1);       // (a thread behind the end copies the last piece too)
    const uint32_t page = piece / pool.units, unit = piece - page * pool.units;
    const uint32_t layer = page / c.n_pairs, pair = page - layer * c.n_pairs;
    char* const in = pool.at + (size_t)layer * pool.layer_bytes + (size_t)unit * sizeof(V);
    held[i] = *reinterpret_cast<const V*>(in + (size_t)c.src[pair] * pool.page_bytes);
    to[i] = in + (size_t)c.dst[pair] * pool.page_bytes;
  }
#pragma unroll
  for (int i = 0; i < COPY_AHEAD; ++i) *reinterpret_cast<V*>(to[i]) = held[i];
}

__global__ void __launch_bounds__(256) copy_pages_kernel(CopyPages c) {
  int p = 0;
  while (p + 1 < c.n_pools && blockIdx.x >= c.pools[p + 1].first_group) ++p;
  const CopyPool pool = c.pools[p];
  if (pool.size == 16) copy_pieces<ptl_u32x4_t>(c, pool);
  else if (pool.size == 4) copy_pieces<uint32_t>(c, pool);
  else copy_pieces<uint8_t>(c, pool);
}

// pools: n_pools times (address, layers, pages, bytes a page) in host memory; src, dst: n page numbers in host memory.
extern "C" int ptl_copy_pages(const long* pools, int n_pools, const int32_t* src, const int32_t* dst, int n, hipStream_t stream) {
  if (n <= 0 || n_pools <= 0) return PTL_OK;
  if (n_pools > POOLS || !pools || !src || !dst) return PTL_ERR_ARG;
  auto size_of = [&](int p) {
    const long both = pools[4 * p] | pools[4 * p + 3];
    return both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : 1;
  };
  long a_pair = 0, pairs = PAIRS;            // the pieces of a launch are counted in 32 bits
  for (int p = 0; p < n_pools; ++p) {
    const long *d = pools + 4 * p, at = d[0], layers = d[1], pages = d[2], bytes = d[3];
    if (!at || layers <= 0 || pages <= 0 || bytes <= 0) return PTL_ERR_ARG;
    for (int i = 0; i < n; ++i)
      if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages) return PTL_ERR_ARG;
    const long one = layers * (bytes / size_of(p));
    if (one >= 1l << 30) return PTL_ERR_ARG;
    a_pair += one + 256 * COPY_AHEAD;
  }
  pairs = min(pairs, max(1l, (1l << 30) / a_pair));
  for (int first = 0; first < n; first += pairs) {
    CopyPages c{};
    c.n_pools = n_pools;
    c.n_pairs = min((int)pairs, n - first);
    uint32_t groups = 0;
    for (int p = 0; p < n_pools; ++p) {
      const long* d = pools + 4 * p;
      CopyPool& pool = c.pools[p];
      pool.at = (char*)d[0];
      pool.page_bytes = d[3];
      pool.layer_bytes = d[2] * d[3];
      pool.size = size_of(p);
      pool.units = (uint32_t)(d[3] / pool.size);
      pool.pieces = (uint32_t)(d[1] * c.n_pairs) * pool.units;
      pool.first_group = groups;
      groups += (pool.pieces + 256 * COPY_AHEAD - 1) / (256 * COPY_AHEAD);
    }
    for (int i = 0; i < c.n_pairs; ++i) { c.src[i] = src[first + i]; c.dst[i] = dst[first + i]; }
    copy_pages_kernel<<<groups, 256, 0, stream>>>(c);
  }
  return ptl_launch_status();
}
