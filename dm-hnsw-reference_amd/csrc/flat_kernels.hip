// Flat scoring kernels for gfx950 (include/shine_gpu.h shine_flat_*): 8-bit row quantisation, the scaled 8-bit matrix
// product of a query batch with a record table, score adjustments, and top-k.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "flat.h"

namespace shine::flat {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// 16 bytes of T at any address that T allows: global memory takes 16-byte accesses at element alignment
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
  T v[N];
};

__device__ inline float to_f32(float x) { return x; }
__device__ inline float to_f32(__half x) { return __half2float(x); }
__device__ inline float to_f32(__hip_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ inline T from_f32(float x);
template <>
__device__ inline float from_f32<float>(float x) { return x; }
template <>
__device__ inline __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ inline __hip_bfloat16 from_f32<__hip_bfloat16>(float x) { return __float2bfloat16(x); }

// ---------------------------------------------------------------------------------------------- quantisation
// scale = f32(max|x| / 127); code = the integer nearest to x / scale in real arithmetic, halves to even.  The quotient
// of 32-bit numbers rounded to 32 bits can land on a half that the real quotient misses, so the integer next to
// x * (1 / scale) is corrected by the sign of the remainder x - code * scale, which one fused multiply-add has exactly
// near scale / 2 (x and code * scale are multiples of a common unit there, their difference a 24-bit multiple of it).
// For scales below 1e-30, where 1 / scale may be infinite, the quotient is taken in 64 bits: it is off by 2^-53, and a
// quotient of 24-bit numbers that is no half is at least 2^-33 from every half.
__device__ inline int code_of(float x, float scale, float inv) {
  float m;
  if (scale >= 1e-30f) {
    m = rintf(x * inv);
    const float e = fmaf(-m, scale, x), e2 = 2.0f * fabsf(e);
    const float step = e > 0.0f ? 1.0f : -1.0f;
    if (e2 > scale || (e2 == scale && (static_cast<int>(m) & 1))) m += step;
  } else {
    m = static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(scale)));
  }
  return static_cast<int>(fminf(fmaxf(m, -127.0f), 127.0f));
}

// One group of G lanes per row, 8 components a lane and step.
template <class T, int G>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a, uint32_t pitch) {
  const uint32_t lane = threadIdx.x % G;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (256 / G) + threadIdx.x / G;
  if (row >= a.n) return;
  const T* src = static_cast<const T*>(a.rows) + row * a.ld;
  uint32_t top = 0;
  for (uint32_t c = lane * 8; c < a.dim; c += G * 8)
    for (uint32_t i = c; i < c + 8 && i < a.dim; ++i) {
      const uint32_t bits = __float_as_uint(to_f32(src[i])) & 0x7FFFFFFFu;
      top = bits > top ? bits : top;
    }
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(top, o, G);
    top = other > top ? other : top;
  }
  const bool finite = top < 0x7F800000u;
  const float scale = finite ? __uint_as_float(top) / 127.0f : __uint_as_float(0x7FC00000u);
  const float inv = 1.0f / scale;
  int squares = 0;
  for (uint32_t c = lane * 8; c < pitch; c += G * 8) {
    uint64_t packed = 0;
    for (uint32_t i = 0; i < 8; ++i) {
      int code = 0;
      if (c + i < a.dim && finite && scale > 0.0f) code = code_of(to_f32(src[c + i]), scale, inv);
      squares += code * code;
      packed |= static_cast<uint64_t>(static_cast<uint8_t>(code)) << (8 * i);
    }
    *reinterpret_cast<uint64_t*>(a.codes + row * pitch + c) = packed;
  }
  for (int o = G / 2; o > 0; o >>= 1) squares += __shfl_xor(squares, o, G);
  if (lane == 0) {
    a.scales[row] = scale;
    if (a.half_norms) a.half_norms[row] = -0.5f * ((static_cast<float>(squares) * scale) * scale);
  }
}

// ---------------------------------------------------------------------------------------------- scores
// out[i][j] = (float(sum_k qc[i][k] * xc[j][k]) * qscale[i]) * scale[j] (+ bias[j]).  Records are the rows and queries
// the columns of the matrix instruction, so that a lane's four sums are neighbours of one output row; tile t's rows
// 4g .. 4g + 3 are records 8g + 4t .. 8g + 4t + 3 of a block of 32, so two tiles give a lane eight neighbours.
template <class T>
__global__ __launch_bounds__(256) void scores_kernel(ScoresArgs a) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t record0 = (static_cast<uint64_t>(blockIdx.x) * 4 + wave) * 32;
  const uint32_t query0 = blockIdx.y * 64;
  if (record0 >= a.n) return;
  const uint32_t col = lane & 15, group = lane >> 4;
  const int8_t* qp[4];
  const int8_t* xp[2];
  for (int i = 0; i < 4; ++i) {  // rows behind the last one read the last one; their sums are not written
    const uint32_t q = query0 + i * 16 + col;
    qp[i] = a.qcodes + static_cast<uint64_t>(q < a.nq ? q : a.nq - 1) * a.pitch + group * 16;
  }
  for (int t = 0; t < 2; ++t) {
    const uint64_t r = record0 + (col >> 2) * 8 + t * 4 + (col & 3);
    xp[t] = a.codes + (r < a.n ? r : a.n - 1) * a.pitch + group * 16;
  }
  v4i acc[4][2] = {};
  for (uint32_t c = 0; c < a.pitch; c += 64) {
    v4i x[2];
    for (int t = 0; t < 2; ++t) x[t] = *reinterpret_cast<const v4i*>(xp[t] + c);
    for (int i = 0; i < 4; ++i) {
      const v4i q = *reinterpret_cast<const v4i*>(qp[i] + c);
      for (int t = 0; t < 2; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t], q, acc[i][t], 0, 0, 0);
    }
  }
  const uint64_t r0 = record0 + group * 8;
  float xs[8], b[8];
  for (int j = 0; j < 8; ++j) {
    const uint64_t r = r0 + j < a.n ? r0 + j : a.n - 1;
    xs[j] = a.scales[r];
    b[j] = a.bias ? a.bias[r] : 0.0f;
  }
  for (int i = 0; i < 4; ++i) {
    const uint32_t q = query0 + i * 16 + col;
    if (q >= a.nq) continue;
    const float qs = a.qscales[q];
    T* dst = static_cast<T*>(a.out) + q * a.ld;
    for (int j = 0; j < 8; ++j) {
      if (r0 + j >= a.n) break;
      float v = (static_cast<float>(acc[i][j >> 2][j & 3]) * qs) * xs[j];
      if (a.bias) v += b[j];
      dst[r0 + j] = from_f32<T>(v);
    }
  }
}

// ---------------------------------------------------------------------------------------------- adjust
// One workgroup per (row, kTile columns): the row's history is counted into LDS for the tile's columns (integer
// additions: any order gives the same counts), then every column is read, changed and written once.
constexpr uint32_t kTile = 4096;

template <class T>
__global__ __launch_bounds__(256) void adjust_kernel(AdjustArgs a) {
  __shared__ uint32_t count[kTile];
  const uint32_t row = blockIdx.y;
  const uint64_t c0 = static_cast<uint64_t>(blockIdx.x) * kTile;
  const uint32_t width = static_cast<uint32_t>(a.n - c0 < kTile ? a.n - c0 : kTile);
  const bool history = a.seen && a.seen_n;
  if (history) {
    for (uint32_t i = threadIdx.x; i < width; i += 256) count[i] = 0;
    __syncthreads();
    const int32_t* seen = a.seen + row * a.seen_ld;
    for (uint32_t i = threadIdx.x; i < a.seen_n; i += 256) {
      const int64_t at = static_cast<int64_t>(seen[i]) - static_cast<int64_t>(a.first + c0);
      if (seen[i] >= 0 && at >= 0 && at < width) atomicAdd(&count[at], 1u);
    }
    __syncthreads();
  }
  const float r = a.repetition ? a.repetition[row] : 1.0f, f = a.frequency ? a.frequency[row] : 0.0f,
              p = a.presence ? a.presence[row] : 0.0f;
  const T* src = static_cast<const T*>(a.scores) + row * a.ld + c0;
  T* dst = static_cast<T*>(a.out) + row * a.out_ld + c0;
  for (uint32_t i = threadIdx.x; i < width; i += 256) {
    const uint64_t record = a.first + c0 + i;
    float v = to_f32(src[i]);
    if (history && count[i]) v = ((v > 0.0f ? v / r : v * r) - f * static_cast<float>(count[i])) - p;
    if (a.bias) v += a.bias[row * a.bias_ld + record];
    if (a.allow && !((a.allow[row * a.allow_ld + (record >> 5)] >> (record & 31)) & 1u)) v = -__builtin_huge_valf();
    dst[i] = from_f32<T>(v);
  }
}

// ---------------------------------------------------------------------------------------------- top-k
// A key holds the value's order in its high word and the id's inverse in its low one: the larger key is the better
// answer and equal values go to the lower id.  Key 0 is no answer; so are -inf and NaN.
__device__ inline uint64_t key_of(float v, uint32_t id) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 orders as +0
  const uint32_t order = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(order) << 32 | (0xFFFFFFFFu - id);
}
__device__ inline float key_value(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ inline int32_t key_id(uint64_t key) {
  return static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

constexpr uint32_t kKeys = 1024;  // keys a workgroup holds: k of them kept, the rest room for newer ones

struct Held {
  uint64_t key[kKeys];
  uint32_t count;
  uint64_t floor;  // the k-th best key held when the room last ran out: smaller keys are no answers
};

// descending, over the first n (a power of two) keys
__device__ inline void sort_keys(uint64_t* key, uint32_t n) {
  for (uint32_t size = 2; size <= n; size <<= 1)
    for (uint32_t step = size >> 1; step > 0; step >>= 1) {
      for (uint32_t i = threadIdx.x; i < n / 2; i += blockDim.x) {
        const uint32_t lo = 2 * step * (i / step) + i % step, hi = lo + step;
        const bool up = (lo & size) != 0;
        const uint64_t x = key[lo], y = key[hi];
        if ((x < y) != up) {
          key[lo] = y;
          key[hi] = x;
        }
      }
      __syncthreads();
    }
}

// Sorts what is held and keeps the best k.  All threads call it, behind a barrier; it ends with one.
__device__ inline void compact(Held& h, uint32_t k) {
  const uint32_t held = h.count < kKeys ? h.count : kKeys;
  uint32_t n = 2;
  while (n < held) n <<= 1;
  for (uint32_t i = held + threadIdx.x; i < n; i += blockDim.x) h.key[i] = 0;
  __syncthreads();
  sort_keys(h.key, n);
  if (threadIdx.x == 0) {
    h.count = held < k ? held : k;
    if (held >= k) h.floor = h.key[k - 1];
  }
  __syncthreads();
}

// Offers each thread's N keys (0: none).  Keys that found no room are offered again behind a compaction, which leaves
// kKeys - k places, so every turn of the loop places some and it ends.
template <int N>
__device__ inline void offer(Held& h, uint32_t k, const uint64_t (&key)[N]) {
  uint32_t pending = 0;
  for (int i = 0; i < N; ++i)
    if (key[i] > h.floor) pending |= 1u << i;
  for (;;) {
    for (int i = 0; i < N; ++i)
      if (pending >> i & 1u) {
        if (key[i] <= h.floor) {
          pending &= ~(1u << i);
        } else {
          const uint32_t at = atomicAdd(&h.count, 1u);
          if (at < kKeys) {
            h.key[at] = key[i];
            pending &= ~(1u << i);
          }
        }
      }
    if (!__syncthreads_or(pending != 0)) return;
    compact(h, k);
  }
}

template <class T>
__device__ inline void write_best(const Held& h, uint32_t k, T* values, int32_t* ids) {
  for (uint32_t i = threadIdx.x; i < k; i += blockDim.x) {
    const bool some = i < h.count;
    values[i] = from_f32<T>(some ? key_value(h.key[i]) : -__builtin_huge_valf());
    ids[i] = some ? key_id(h.key[i]) : -1;
  }
}

template <class T>
__global__ __launch_bounds__(256) void topk_kernel(TopkArgs a, bool to_keys) {
  __shared__ Held h;
  constexpr int N = 8;
  const uint32_t row = blockIdx.y, slice = blockIdx.x;
  if (threadIdx.x == 0) {
    h.count = 0;
    h.floor = 0;
  }
  __syncthreads();
  const T* src = static_cast<const T*>(a.scores) + row * a.ld;
  const uint64_t per = (a.n + a.slices - 1) / a.slices, c0 = slice * per, c1 = c0 + per < a.n ? c0 + per : a.n;
  for (uint64_t c = c0; c < c1; c += 256 * N) {
    uint64_t key[N];
    for (int i = 0; i < N; ++i) {
      const uint64_t at = c + i * 256 + threadIdx.x;
      key[i] = 0;
      if (at < c1) {
        const float v = to_f32(src[at]);
        if (v >= -3.402823466e38f) key[i] = key_of(v, static_cast<uint32_t>(a.first + at));
      }
    }
    offer(h, a.k, key);
  }
  compact(h, a.k);
  if (to_keys) {
    uint64_t* out = a.keys + (static_cast<uint64_t>(row) * a.key_ld + slice) * a.k;
    for (uint32_t i = threadIdx.x; i < a.k; i += 256) out[i] = i < h.count ? h.key[i] : 0;
  } else {
    write_best(h, a.k, static_cast<T*>(a.values) + static_cast<uint64_t>(row) * a.k,
               a.ids + static_cast<uint64_t>(row) * a.k);
  }
}

template <class T>
__global__ __launch_bounds__(256) void merge_kernel(MergeArgs a) {
  __shared__ Held h;
  constexpr int N = 4;
  const uint32_t row = blockIdx.x;
  if (threadIdx.x == 0) {
    h.count = 0;
    h.floor = 0;
  }
  __syncthreads();
  const uint64_t* src = a.keys + row * a.count;
  for (uint64_t c = 0; c < a.count; c += 256 * N) {
    uint64_t key[N];
    for (int i = 0; i < N; ++i) {
      const uint64_t at = c + i * 256 + threadIdx.x;
      key[i] = at < a.count ? src[at] : 0;
    }
    offer(h, a.k, key);
  }
  compact(h, a.k);
  write_best(h, a.k, static_cast<T*>(a.values) + static_cast<uint64_t>(row) * a.k,
             a.ids + static_cast<uint64_t>(row) * a.k);
}

}  // namespace

#define SHINE_BY_ELEM(elem, CALL)                 \
  switch (elem) {                                 \
    case kF32: { using T = float; CALL; break; }  \
    case kF16: { using T = __half; CALL; break; } \
    case kBF16: { using T = __hip_bfloat16; CALL; break; } \
    default: return hipErrorInvalidValue;         \
  }

hipError_t launch_quantize(int elem, const QuantizeArgs& a, hipStream_t s) {
  const uint32_t pitch = code_pitch(a.dim);
#define SHINE_GROUP(GG)                                                                                    \
  hipLaunchKernelGGL((quantize_kernel<T, GG>), dim3(static_cast<uint32_t>((a.n + 256 / GG - 1) / (256 / GG))), \
                     dim3(256), 0, s, a, pitch)
  SHINE_BY_ELEM(elem, if (pitch <= 64) SHINE_GROUP(8); else if (pitch <= 128) SHINE_GROUP(16);
                else if (pitch <= 256) SHINE_GROUP(32); else SHINE_GROUP(64));
#undef SHINE_GROUP
  return hipGetLastError();
}

hipError_t launch_scores(int out_elem, const ScoresArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>((a.n + 127) / 128), (a.nq + 63) / 64);
  SHINE_BY_ELEM(out_elem, hipLaunchKernelGGL(scores_kernel<T>, grid, dim3(256), 0, s, a));
  return hipGetLastError();
}

hipError_t launch_adjust(int elem, const AdjustArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>((a.n + kTile - 1) / kTile), a.nq);
  SHINE_BY_ELEM(elem, hipLaunchKernelGGL(adjust_kernel<T>, grid, dim3(256), 0, s, a));
  return hipGetLastError();
}

uint32_t topk_slices(uint32_t nq, uint64_t n) {
  const uint64_t want = (1024 + nq - 1) / nq, most = (n + 4095) / 4096;
  const uint64_t s = want < most ? want : most;
  return static_cast<uint32_t>(s ? s : 1);
}

hipError_t launch_topk(int elem, bool keys_only, const TopkArgs& a, hipStream_t s) {
  const bool to_keys = keys_only || a.slices > 1;
  SHINE_BY_ELEM(elem, hipLaunchKernelGGL(topk_kernel<T>, dim3(a.slices, a.nq), dim3(256), 0, s, a, to_keys));
  return hipGetLastError();
}

hipError_t launch_merge(int elem, const MergeArgs& a, hipStream_t s) {
  SHINE_BY_ELEM(elem, hipLaunchKernelGGL(merge_kernel<T>, dim3(a.nq), dim3(256), 0, s, a));
  return hipGetLastError();
}

}  // namespace shine::flat
