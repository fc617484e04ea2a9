// Flat scoring kernels for gfx950 (include/shine_gpu.h shine_flat_*): 8-bit row quantisation, the scaled 8-bit matrix
// product of a query batch with a record table, score adjustments, and top-k.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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
__device__ inline float to_f32(__bf16 x) { return static_cast<float>(x); }
template <class T>
__device__ inline T from_f32(float x);
template <>
__device__ inline float from_f32<float>(float x) { return x; }
template <>
__device__ inline __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ inline __bf16 from_f32<__bf16>(float x) { return static_cast<__bf16>(x); }

// ---------------------------------------------------------------------------------------------- quantisation
// scale = f32(max|x| / 127); code = the integer nearest to x / scale in real arithmetic, halves to even.  The quotient
// of 32-bit numbers rounded to 32 bits can land on a half that the real quotient misses, so the integer next to
// x * (1 / scale) is corrected by the sign of the remainder x - code * scale, which one fused multiply-add has exactly
// near scale / 2 (x and code * scale are multiples of a common unit there, their difference a 24-bit multiple of it).
// For scales below 1e-30, where 1 / scale may be infinite, the quotient is taken in 64 bits: it is off by 2^-53, and a
// quotient of 24-bit numbers that is no half is at least 2^-33 from every half.
struct Scale {
  float scale, inv, near;
  bool some;  // the row has codes other than 0
  __device__ explicit Scale(uint32_t top) {  // the largest magnitude's bits
    const bool finite = top < 0x7F800000u;
    scale = finite ? __uint_as_float(top) / 127.0f : __uint_as_float(0x7FC00000u);
    some = finite && scale > 0.0f;
    inv = 1.0f / scale;
    near = scale * 0.4999995f;
  }
  __device__ int code(float x) const {
    if (!some) return 0;
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
  // Four codes in a word.  A remainder below `near` needs no correction and its integer no clamp (|x| <= the largest), so the
  // four are corrected together or, nearly always, not at all: seven operations a component instead of about fifty.
  __device__ uint32_t codes(const float* x) const {
    uint32_t packed = 0;
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = rintf(x[i] * inv);
      worst = fmaxf(worst, fabsf(fmaf(-m, scale, x[i])));
      packed = __builtin_amdgcn_cvt_pk_u8_f32(m + 128.0f, i, packed);
    }
    packed ^= 0x80808080u;
    if (!some || !(worst < near) || scale < 1e-30f) {
      packed = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) packed |= (static_cast<uint32_t>(code(x[i])) & 0xFFu) << (8 * i);
    }
    return packed;
  }
};

// V = 16 bytes of components that a lane takes in a step; components behind dim are 0
template <class T, int V>
__device__ inline void load_components(float (&x)[V], const T* src, uint32_t c, uint32_t dim) {
  if (c + V <= dim) {
    const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(src + c);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f32(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = c + i < dim ? to_f32(src[c + i]) : 0.0f;
  }
}

// G lanes per row and S steps of 16 bytes a lane, held in registers between the maximum and the codes (S = 0: rows too wide
// for that are read twice).  A group takes R rows a turn and asks for the next turn's before it looks at this one's.  Bound by
// HBM: 1M x 128 f32 takes 133 us, 4.8 TB/s, where a copy reaches 5.1; one row a turn takes 181 to 216, four rows 184, and
// of 1,024 .. 8,192 workgroups and one for every turn 8,192 are best or near it for each width and type.
template <class T, int G, int S, int R>
__global__ __launch_bounds__(256) void quantize_kernel(QuantizeArgs a, uint32_t pitch) {
  constexpr int V = 16 / sizeof(T), H = S ? S : 1;
  constexpr uint32_t kRows = 256 / G * R;  // of a workgroup's turn
  const uint32_t lane = threadIdx.x % G;
  float next[R][H][V];
  auto fetch = [&](uint64_t row0) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const T* src = static_cast<const T*>(a.rows) + min(row0 + k * (256 / G), a.n - 1) * a.ld;
#pragma unroll
      for (int j = 0; j < H; ++j) load_components<T, V>(next[k][j], src, (j * G + lane) * V, a.dim);
    }
  };
  uint64_t row0 = static_cast<uint64_t>(blockIdx.x) * kRows + threadIdx.x / G;
  if (S) fetch(row0);
  for (; row0 < a.n; row0 += static_cast<uint64_t>(gridDim.x) * kRows) {
    float x[R][H][V];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int j = 0; j < H; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) x[k][j][i] = next[k][j][i];
    if (S) fetch(row0 + static_cast<uint64_t>(gridDim.x) * kRows);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const uint64_t row = row0 + k * (256 / G);
      if (row >= a.n) break;
      const T* src = static_cast<const T*>(a.rows) + row * a.ld;
      uint32_t top = 0;
      auto raise = [&top](const float(&v)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
      };
      if (S) {
#pragma unroll
        for (int j = 0; j < H; ++j) raise(x[k][j]);
      } else {
        for (uint32_t c = lane * V; c < a.dim; c += G * V) {
          load_components<T, V>(x[0][0], src, c, a.dim);
          raise(x[0][0]);
        }
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, G)));
      const Scale s(top);
      int squares = 0;
      auto write = [&](const float(&v)[V], uint32_t c) {
        uint32_t packed[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          packed[i] = s.codes(v + i * 4);
          squares = __builtin_amdgcn_sdot4(static_cast<int>(packed[i]), static_cast<int>(packed[i]), squares, false);
        }
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.codes + row * pitch + c);
        if (V == 4) *dst = packed[0];
        else *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[V / 4 - 1]);
      };
      if (S) {
#pragma unroll
        for (int j = 0; j < H; ++j)
          if ((j * G + lane) * V < pitch) write(x[k][j], (j * G + lane) * V);
      } else {
        for (uint32_t c = lane * V; c < pitch; c += G * V) {
          load_components<T, V>(x[0][0], src, c, a.dim);
          write(x[0][0], c);
        }
      }
      if (a.half_norms)
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) squares += __shfl_xor(squares, o, G);
      if (lane == 0) {
        a.scales[row] = s.scale;
        if (a.half_norms) a.half_norms[row] = -0.5f * ((static_cast<float>(squares) * s.scale) * s.scale);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- products
// Records are the rows and queries the columns of the matrix instruction, so that a lane's four sums are neighbours of
// one output row; tile t's rows 4g .. 4g + 3 are records 8g + 4t .. 8g + 4t + 3 of a block of 32, so two tiles give a
// lane eight neighbours: records 8 (lane / 16) .. + 7 of the block for query lane % 16 of the tile.
//
// Rows of at most 256 codes (kStreamPitch): a wave keeps the codes of QT * 16 queries in registers and streams blocks of
// records past them, so nothing passes through LDS and a record is read once for all of the wave's queries.  The sums
// start at kMagic: |sum| <= 256 * 127^2 < 2^22, so kMagic + sum read as a float is 1.5 * 2^23 + sum, with no conversion.
constexpr uint32_t kStreamPitch = 256;
constexpr int kMagic = 0x4B400000;
constexpr float kMagicF = 12582912.0f;

template <int KC>
struct Block {  // a wave's 32 records
  v4i x[2][KC];
};

// The wave's number, in a scalar register: what follows from it alone is computed once for the wave
__device__ inline uint32_t wave_number() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Between a wave's own writes to LDS and its lanes' reads of them (a wave's LDS accesses are in order: no wait)
__device__ inline void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// PAIRED: a lane's eight sums are neighbours (above); else tile t holds records 16 t .. 16 t + 15 and a lane four neighbours
// of each tile: the better order for writing 32-bit scores, 64 bytes of a row an instruction.
template <int KC, bool PAIRED = true>
__device__ inline void load_block(Block<KC>& b, const int8_t* codes, uint64_t record0, uint64_t n) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
  const int8_t* p = codes + record0 * (KC * 64);
  const uint32_t last = n - record0 < 32 ? static_cast<uint32_t>(n - record0) - 1 : 31;
#pragma unroll
  for (int t = 0; t < 2; ++t) {  // rows behind the last one read the last one; nobody uses their sums
    const uint32_t at = min(PAIRED ? (col >> 2) * 8 + t * 4 + (col & 3) : t * 16 + col, last) * (KC * 64) + group * 16;
#pragma unroll
    for (int c = 0; c < KC; ++c) b.x[t][c] = *reinterpret_cast<const v4i*>(p + at + c * 64);
  }
}

template <int KC, int QT>
__device__ inline void load_queries(v4i (&q)[QT][KC], const int8_t* qcodes, uint32_t query0, uint32_t nq) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const uint32_t at = query0 + i * 16 + (lane & 15);
    const int8_t* p = qcodes + static_cast<uint64_t>(at < nq ? at : nq - 1) * (KC * 64) + (lane >> 4) * 16;
#pragma unroll
    for (int c = 0; c < KC; ++c) q[i][c] = *reinterpret_cast<const v4i*>(p + c * 64);
  }
}

// kMagic four times, in registers of its own that the compiler does not fill anew for every product
__device__ inline v4i magic_start() {
  v4i m = {kMagic, kMagic, kMagic, kMagic};
  asm volatile("" : "+v"(m));
  return m;
}

template <int KC>
__device__ inline void sums(const Block<KC>& b, const v4i (&q)[KC], const v4i& start, float (&f)[8]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    v4i acc = start;
#pragma unroll
    for (int c = 0; c < KC; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b.x[t][c], q[c], acc, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[t * 4 + j] = __int_as_float(acc[j]);
  }
}

// Workgroups of one record range and all query blocks run on one XCD (workgroup b runs on XCD b % 8), so that its L2
// serves the range to all of them.
struct Place {
  uint32_t query_block, range;
};
__device__ inline Place place_of(uint32_t query_blocks) {
  const uint32_t xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
  return {i % query_blocks, (i / query_blocks) * 8 + xcd};
}

// ---------------------------------------------------------------------------------------------- scores
// out[i][j] = (float(sum_k qc[i][k] * xc[j][k]) * qscale[i]) * scale[j] (+ bias[j])
template <class T, int N>
__device__ inline void store_scores(T* dst, const float* v) {
  Vec<T, N> o;
#pragma unroll
  for (int j = 0; j < N; ++j) o.v[j] = from_f32<T>(v[j]);
  *reinterpret_cast<Vec<T, N>*>(dst) = o;
}

// Where a lane's j-th sum of a block belongs, and the writing of all eight to a row, from the block's first record on.
template <class T>
struct Order {
  static constexpr bool kPaired = sizeof(T) == 2;
  __device__ static uint32_t record(uint32_t group, int j) {
    return kPaired ? group * 8 + j : (j >> 2) * 16 + group * 4 + (j & 3);
  }
  __device__ static void store(T* row, uint32_t group, const float (&v)[8]) {
    if (kPaired) {
      store_scores<T, 8>(row + group * 8, v);
    } else {
      store_scores<T, 4>(row + group * 4, v);
      store_scores<T, 4>(row + 16 + group * 4, v + 4);
    }
  }
  __device__ static void store(T* row, uint32_t group, const float (&v)[8], uint32_t left) {  // the row's last `left` records
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (record(group, j) < left) row[record(group, j)] = from_f32<T>(v[j]);
  }
};

// The next block's codes, scales and biases are asked for before this block's scores are written, and no branch is around
// the writes: memory accesses end in order, so what waits for a load must know how many writes are behind it.  Lanes
// whose query is behind the last one hold the last one and write its scores once more; the block that the records end in
// comes last, on its own.  Bound by reading the codes: 1 x 1M x 128, 24 us, 5.6 TB/s.
//
// E (not void): the queries' element type; each wave quantises its 16 queries itself, which saves a launch where few blocks
// follow (1 x 10,000 x 128: 8.7 us a call against 15.0).
template <class E>
__device__ inline void quantize_fragment(v4i& codes, const Scale& s, const float (&x)[16]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) codes[w] = static_cast<int>(s.codes(x + w * 4));
}

template <class T, int KC, int QT, class E>
__global__ __launch_bounds__(256) void scores_stream_kernel(ScoresArgs a, uint64_t per_range) {
  __shared__ float beside[4][2][32];  // each wave's records' scales and biases
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 15, group = lane >> 4;
  const uint64_t blocks = (a.n + 31) / 32, whole = a.n / 32, b0 = blockIdx.x * per_range,
                 b1 = b0 + per_range < blocks ? b0 + per_range : blocks;
  if (b0 + wave >= b1) return;
  v4i q[QT][KC];
  float qs[QT];
  T* to[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const uint32_t r = min(i * 16 + col, a.nq - 1);
    to[i] = static_cast<T*>(a.out) + r * a.ld;
    if constexpr (std::is_void_v<E>) {
      qs[i] = a.qscales[r];
    } else {
      constexpr int V = 16 / sizeof(E);
      const E* src = static_cast<const E*>(a.queries) + r * a.queries_ld;
      float x[KC][16];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int h = 0; h < 16; h += V) {
          float part[V];
          load_components<E, V>(part, src, c * 64 + group * 16 + h, a.dim);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[c][h + j] = part[j];
            top = max(top, __float_as_uint(part[j]) & 0x7FFFFFFFu);
          }
        }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      const Scale s(top);
      qs[i] = s.scale;
#pragma unroll
      for (int c = 0; c < KC; ++c) quantize_fragment<E>(q[i][c], s, x[c]);
    }
  }
  if constexpr (std::is_void_v<E>) load_queries<KC, QT>(q, a.qcodes, 0, a.nq);
  const v4i start = magic_start();
  const float* biases = a.bias ? a.bias : a.scales;
  Block<KC> next;
  float next_xs, next_bias;
  auto fetch = [&](uint64_t b) {
    load_block<KC, Order<T>::kPaired>(next, a.codes, b * 32, a.n);
    const uint64_t r = b * 32 + (lane & 31), from = r < a.n ? r : a.n - 1;
    next_xs = a.scales[from];
    next_bias = biases[from];
  };
  Block<KC> x;
  auto stage = [&] {  // what was fetched is next to be scored: here, and not where the compiler would first need it
    x = next;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < KC; ++c) asm volatile("" : "+v"(x.x[t][c]));
    if (lane < 32) {
      beside[wave][0][lane] = next_xs;
      beside[wave][1][lane] = a.bias ? next_bias : -0.0f;  // adding -0 changes nothing
    }
    wave_sync();
  };
  float xs[8], bias[8];
  auto look = [&] {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xs[j] = beside[wave][0][Order<T>::record(group, j)];
      bias[j] = beside[wave][1][Order<T>::record(group, j)];
    }
    wave_sync();
  };
  auto score = [&](int i, float(&v)[8]) {
    sums<KC>(x, q[i], start, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ((v[j] - kMagicF) * qs[i]) * xs[j] + bias[j];
  };
  uint64_t b = b0 + wave;
  fetch(b);
  stage();
  for (; b < b1 && b < whole; b += 4) {
    look();
    fetch(b + 4 < b1 ? b + 4 : b1 - 1);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float v[8];
      score(i, v);
      Order<T>::store(to[i] + b * 32, group, v);
    }
    stage();  // at the end: at the start, where the first block's loads have no writes behind them, it would wait for all
  }
  if (b < b1) {
    look();
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float v[8];
      score(i, v);
      Order<T>::store(to[i] + b * 32, group, v, static_cast<uint32_t>(a.n - b * 32));
    }
  }
}

// More than 32 queries write more than they read: 128-byte lines of the rows, each whole and by one instruction, whatever the
// rows' starts.  Lines written in parts cost the memory a read and a write each where a part is evicted before the other comes
// (rows of 100,003 f32 in the streams above: 8.05M write requests, 0.85M of them partial, for 6.4M lines' halves).  A wave keeps
// QT * 16 queries and goes through neighbouring records, a line's number of them a turn.  Queries are the products' rows, so
// that a lane has its record's scale and bias in registers and sums of four queries.  A row's scores go into a ring of two lines
// in LDS, at the offsets that they have in memory's lines; what completes a line is written, the rest is there for the next
// turn.  Rings of 16 queries are turned against one another so that the 64 lanes of a write, and of a read, meet different banks.
//
// A run's first line begins in the records before: long runs of f32 score them again (a turn more of 8 or more lines), short ones
// and 16-bit scores, whose turns are twice as long, write the line's part.  Memory accesses end in order, so a turn's end, where
// the next turn's codes are taken, waits for the writes of the turn before it: P lines a turn, two where the registers have room
// for their codes, put that off (100 us a call against 106).
//
// 1024 x 100,003 x 96, kernel and quantising: f32 166 -> 100 us (with lines' parts written 119), bf16 into four buffers by turns
// 97 -> 78 (into one, which the caches half hold, 77 -> 58); rows of 100,000: 114 -> 102, 74 -> 72 (47 -> 54).  128 queries a wave:
// 130; 32, with four waves a SIMD: 125.  What bounds it is the writing: 4.4 TB/s, of 6.7 that a fill reaches.
template <class T, int KC, int QT, int P>
__global__ __launch_bounds__(256, 2) void scores_lines_kernel(ScoresArgs a, uint32_t query_blocks, uint64_t per) {
  constexpr uint32_t kLine = 128 / sizeof(T), kPiece = 16 / sizeof(T);  // scores of a line and of 16 bytes
  constexpr int NT = kLine / 16, U = QT * 2;
  const bool again = sizeof(T) == 4 && per >= 8;
  __shared__ __attribute__((aligned(16))) uint8_t rings[4][QT * 16][256];
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 15, group = lane >> 4;
  const Place at = place_of(query_blocks);
  const uint32_t query0 = at.query_block * QT * 16;
  const uint64_t lines = (a.n + kLine - 1) / kLine, first = (at.range * 4ull + wave) * per, end = min(first + per, lines);
  if (first >= end) return;
  uint8_t* ring = &rings[wave][0][0];
  T* out = static_cast<T*>(a.out);
  auto row_of = [&](uint32_t r) { return out + min(query0 + r, a.nq - 1) * a.ld; };
  auto turned = [](uint32_t r) { return (r & 1) * 128 + (r >> 2 & 3) * 64; };
  v4i q[QT][KC];
  load_queries<KC, QT>(q, a.qcodes, query0, a.nq);
  float qs[QT][4];
  uint32_t place[QT];  // a byte each for four rows: where in their rings column 0 of an even block's first tile goes
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    place[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t r = i * 16 + group * 4 + j;
      qs[i][j] = a.qscales[min(query0 + r, a.nq - 1)];
      const uint32_t shift = reinterpret_cast<uint64_t>(row_of(r)) & 127;
      place[i] |= ((turned(r) + shift + col * sizeof(T)) & 255) << (8 * j);
    }
  }
  uint64_t line[U];  // where the line goes that holds the first score of a row
#pragma unroll
  for (int u = 0; u < U; ++u) line[u] = (reinterpret_cast<uint64_t>(row_of(u * 8 + (lane >> 3))) & ~127ull) + (lane & 7) * 16;
  const v4i start = magic_start();
  const float* biases = a.bias ? a.bias : a.scales;
  const bool biased = a.bias;
  v4i next[P][NT][KC], x[P][NT][KC];
  float next_xs[P][NT], next_bias[P][NT], xs[P][NT], bias[P][NT];
  auto fetch = [&](uint64_t b0) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint64_t b = min(b0 + p, lines - 1);
      const int8_t* from = a.codes + b * (kLine * KC * 64);
      const uint32_t last = static_cast<uint32_t>(min(a.n - b * kLine, static_cast<uint64_t>(kLine))) - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t r = min(t * 16 + col, last);
#pragma unroll
        for (int c = 0; c < KC; ++c) next[p][t][c] = *reinterpret_cast<const v4i*>(from + r * (KC * 64) + group * 16 + c * 64);
        next_xs[p][t] = (a.scales + b * kLine)[r];
        next_bias[p][t] = (biases + b * kLine)[r];
      }
    }
  };
  auto stage = [&] {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          x[p][t][c] = next[p][t][c];
          asm volatile("" : "+v"(x[p][t][c]));
        }
        xs[p][t] = next_xs[p][t];
        bias[p][t] = biased ? next_bias[p][t] : -0.0f;
        asm volatile("" : "+v"(xs[p][t]), "+v"(bias[p][t]));
      }
  };
  auto score = [&](int p, uint32_t parity) {
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        v4i acc = start;
#pragma unroll
        for (int c = 0; c < KC; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[i][c], x[p][t][c], acc, 0, 0, 0);
        const uint32_t to = ((place[i] & 0x7F7F7F7Fu) + t * 16 * sizeof(T) * 0x01010101u) ^ (place[i] & 0x80808080u) ^ parity * 0x01010101u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<T*>(ring + (i * 16 + group * 4 + j) * 256 + (to >> (8 * j) & 255)) =
              from_f32<T>(((__int_as_float(acc[j]) - kMagicF) * qs[i][j]) * xs[p][t] + bias[p][t]);
      }
    wave_sync();
  };
  auto ring_piece = [&](uint32_t r, uint32_t parity) { return ring + r * 256 + ((turned(r) + parity + (lane & 7) * 16) & 255); };
  // the scores [from, to) of line b: pieces of 16 bytes, or one by one where a piece is not all of these
  auto edge = [&](uint64_t b, uint32_t parity, uint64_t from, uint64_t to) {
#pragma unroll 2
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t r = u * 8 + (lane >> 3);
      T* row = row_of(r);
      const int64_t at = static_cast<int64_t>(b * kLine) + (lane & 7) * kPiece - (reinterpret_cast<uint64_t>(row) & 127) / sizeof(T);
      const Vec<T, kPiece> v = *reinterpret_cast<const Vec<T, kPiece>*>(ring_piece(r, parity));
      const int64_t low = from, high = to;
      if (at >= low && at + kPiece <= high) {
        *reinterpret_cast<Vec<T, kPiece>*>(row + at) = v;
      } else if (at + kPiece > low && at < high) {
#pragma unroll
        for (uint32_t e = 0; e < kPiece; ++e)
          if (at + e >= low && at + e < high) row[at + e] = v.v[e];
      }
    }
  };
  const uint64_t b0 = again && first ? first - P : first, from = again ? 0 : first * kLine,
                 whole = again ? max(first, 1ul) : first + 1;  // the first line that is all of this run's
  auto parity_of = [&](uint64_t b, int p) { return P == 2 ? p * 128u : static_cast<uint32_t>(b - b0 & 1) * 128u; };
  fetch(b0);
  stage();
  for (uint64_t b = b0; b < end; b += P) {
    fetch(b + P);
    if (b >= whole && b + P < lines) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        score(p, parity_of(b, p));
#pragma unroll
        for (int u = 0; u < U; ++u)
          *reinterpret_cast<v4i*>(line[u] + (b + p) * 128) = *reinterpret_cast<const v4i*>(ring_piece(u * 8 + (lane >> 3), parity_of(b, p)));
        wave_sync();
      }
      stage();  // in each branch: behind them both it would wait for all writes
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (b + p + 1 >= first && b + p < end) {
          score(p, parity_of(b, p));
          if (b + p >= first) edge(b + p, parity_of(b, p), from, a.n);
          wave_sync();
        }
      stage();
    }
  }
  if (!again || end == lines) edge(end, static_cast<uint32_t>(end - b0 & 1) * 128, from, min(end * kLine, a.n));
}

// Wider rows: tiles of 256 records x 128 queries, four waves of 128 x 64 each, 64 codes of every row a step.  A step's codes go
// through LDS (a wave reads 12 fragments for 32 matrix instructions) in two buffers; the step after the next is on its way in
// registers meanwhile.  A row's four 16-byte pieces are rotated by its number, so that the 8 rows that one LDS cycle serves
// lie in different banks.  2048 x 32,768 x 1024 with bf16 scores: 89 us, 1.54 POP/s of the 2.06 that a large library product
// reaches; the matrix unit is busy a third of the time, the waves wait for the step's barrier and loads.
constexpr uint32_t kTileRecords = 256, kTileQueries = 128;

struct WideTile {
  int8_t x[2][kTileRecords * 64], q[2][kTileQueries * 64];
};

__device__ inline uint32_t record_piece(uint32_t row, uint32_t piece) {  // rows met together: 0 .. 3 and 8 .. 11 (+ 4)
  return row * 64 + (piece ^ ((row >> 1 & 1) | (row >> 2 & 2))) * 16;
}
__device__ inline uint32_t query_piece(uint32_t row, uint32_t piece) { return row * 64 + (piece ^ (row >> 1 & 3)) * 16; }

// acc[i][t]: query tile i (16 queries) of the wave's four, record tile t of its eight (two to a block of 32)
template <bool PAIRED>
__device__ inline void wide_sums(WideTile& w, const int8_t* codes, uint64_t n, const int8_t* qcodes, uint32_t nq, uint32_t pitch,
                                 uint64_t record0, uint32_t query0, v4i (&acc)[4][8]) {
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 15, group = lane >> 4;
  const int8_t* xbase = codes + record0 * pitch;
  const int8_t* qbase = qcodes + static_cast<uint64_t>(query0) * pitch;
  const uint32_t xlast = static_cast<uint32_t>(min(n - record0, static_cast<uint64_t>(kTileRecords))) - 1,
                 qlast = min(nq - query0, kTileQueries) - 1;
  const uint32_t row = threadIdx.x >> 2, piece = threadIdx.x & 3;  // this thread brings piece `piece` of rows row + 64 j
  uint32_t xat[4], qat[2];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) xat[j] = min(row + 64 * j, xlast) * pitch + piece * 16;  // behind the last row: the last row
#pragma unroll
  for (uint32_t j = 0; j < 2; ++j) qat[j] = min(row + 64 * j, qlast) * pitch + piece * 16;
  v4i xr[4], qr[2];
  auto fetch = [&](uint32_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) xr[j] = *reinterpret_cast<const v4i*>(xbase + xat[j] + c);
#pragma unroll
    for (int j = 0; j < 2; ++j) qr[j] = *reinterpret_cast<const v4i*>(qbase + qat[j] + c);
  };
  auto put = [&](uint32_t buffer) {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) *reinterpret_cast<v4i*>(&w.x[buffer][record_piece(row + 64 * j, piece)]) = xr[j];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) *reinterpret_cast<v4i*>(&w.q[buffer][query_piece(row + 64 * j, piece)]) = qr[j];
  };
  const uint32_t x0 = (wave & 1) * 128, q0 = (wave >> 1) * 64;
  uint32_t xlds[8], qlds[4];
#pragma unroll
  for (uint32_t t = 0; t < 8; ++t) xlds[t] = record_piece(x0 + (t >> 1) * 32 + (PAIRED ? (col >> 2) * 8 + (t & 1) * 4 + (col & 3) : (t & 1) * 16 + col), group);
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) qlds[i] = query_piece(q0 + i * 16 + col, group);
  fetch(0);
  put(0);
  if (pitch > 64) fetch(64);
  __syncthreads();
  for (uint32_t c = 0, buffer = 0; c < pitch; c += 64, buffer ^= 1) {
    v4i xf[8], qf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const v4i*>(&w.q[buffer][qlds[i]]);
#pragma unroll
    for (int t = 0; t < 8; ++t) xf[t] = *reinterpret_cast<const v4i*>(&w.x[buffer][xlds[t]]);
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[t], qf[i], acc[i][t], 0, 0, 0);
    if (c + 64 < pitch) {
      put(buffer ^ 1);  // everyone read it before the last barrier
      if (c + 128 < pitch) fetch(c + 128);
      __syncthreads();
    }
  }
}

template <class T>
__global__ __launch_bounds__(256, 2) void scores_wide_kernel(ScoresArgs a, uint32_t query_blocks, uint32_t record_blocks) {
  __shared__ WideTile w;
  __shared__ float scales[kTileRecords], biases[kTileRecords], qscales[kTileQueries];
  const Place at = place_of(query_blocks);
  if (at.range >= record_blocks) return;
  const uint64_t record0 = static_cast<uint64_t>(at.range) * kTileRecords;
  const uint32_t query0 = at.query_block * kTileQueries;
  {
    const uint64_t r = min(record0 + threadIdx.x, a.n - 1);
    scales[threadIdx.x] = a.scales[r];
    biases[threadIdx.x] = a.bias ? a.bias[r] : -0.0f;  // adding -0 changes nothing
    if (threadIdx.x < kTileQueries) qscales[threadIdx.x] = a.qscales[min(query0 + threadIdx.x, a.nq - 1)];
  }
  v4i acc[4][8] = {};
  wide_sums<Order<T>::kPaired>(w, a.codes, a.n, a.qcodes, a.nq, a.pitch, record0, query0, acc);
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 15, group = lane >> 4;
  const bool whole = record0 + kTileRecords <= a.n;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t at0 = (wave & 1) * 128 + p * 32;
    const uint64_t r0 = record0 + at0;
    float xs[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xs[j] = scales[at0 + Order<T>::record(group, j)];
      b[j] = biases[at0 + Order<T>::record(group, j)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = (wave >> 1) * 64 + i * 16 + col;
      const float qs = qscales[q];
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (static_cast<float>(acc[i][p * 2 + (j >> 2)][j & 3]) * qs) * xs[j] + b[j];
      // queries behind the last one are the last one: its scores are written once more
      T* row = static_cast<T*>(a.out) + min(query0 + q, a.nq - 1) * a.ld + r0;
      if (whole) Order<T>::store(row, group, v);
      else if (r0 < a.n) Order<T>::store(row, group, v, static_cast<uint32_t>(min(a.n - r0, static_cast<uint64_t>(32))));
    }
  }
}

// Wide rows, few queries: every wave 32 records, the queries' codes from the caches.
template <class T>
__global__ __launch_bounds__(256) void scores_few_kernel(ScoresArgs a) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
  const uint64_t record0 = (static_cast<uint64_t>(blockIdx.x) * 4 + wave_number()) * 32;
  if (record0 >= a.n) return;
  const uint32_t last = static_cast<uint32_t>(min(a.n - record0, 32ul)) - 1;
  const int8_t* xbase = a.codes + record0 * a.pitch;
  uint32_t xat[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) xat[t] = min(Order<T>::kPaired ? (col >> 2) * 8 + t * 4 + (col & 3) : t * 16 + col, last) * a.pitch + group * 16;
  const uint32_t qat = min(col, a.nq - 1) * a.pitch + group * 16;
  v4i acc[2] = {};
  auto step = [&](const v4i(&x)[2], uint32_t c) {
    const v4i q = *reinterpret_cast<const v4i*>(a.qcodes + qat + c);
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t], q, acc[t], 0, 0, 0);
  };
  uint32_t c = 0;
  for (; c + 256 <= a.pitch; c += 256) {  // four steps' records are asked for together
    v4i x[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int t = 0; t < 2; ++t) x[k][t] = *reinterpret_cast<const v4i*>(xbase + xat[t] + c + k * 64);
#pragma unroll
    for (int k = 0; k < 4; ++k) step(x[k], c + k * 64);
  }
  for (; c < a.pitch; c += 64) {
    v4i x[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) x[t] = *reinterpret_cast<const v4i*>(xbase + xat[t] + c);
    step(x, c);
  }
  float xs[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint64_t r = min(record0 + Order<T>::record(group, j), a.n - 1);
    xs[j] = a.scales[r];
    b[j] = a.bias ? a.bias[r] : -0.0f;
  }
  const uint32_t q = min(col, a.nq - 1);  // behind the last query: the last one once more
  const float qs = a.qscales[q];
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (static_cast<float>(acc[j >> 2][j & 3]) * qs) * xs[j] + b[j];
  T* row = static_cast<T*>(a.out) + q * a.ld + record0;
  if (last == 31) Order<T>::store(row, group, v);
  else Order<T>::store(row, group, v, last + 1);
}

// ---------------------------------------------------------------------------------------------- adjust
// One workgroup per (row, TILE columns).  The row's history is counted in LDS for the tile's columns, in 16 bits beside a bit
// for each column that is met (integer additions: any order gives the same counts).  Then every column is read, changed
// and written once, 16 bytes a lane.  Tiles start at multiples of 32 records, so a lane's columns share a word of allowed
// bits and one of met ones.
// Two steps' loads are asked for before anything of them is written (memory accesses end in order), the first two before the
// history is counted.  256 x 151,937 bf16 with histories of 2,048 and masks: 45 us, 3.6 TB/s, and 42 without the histories; four
// steps' loads take the registers of every third wave (56 us), tiles of 4,096 columns read the histories twice (47; but 141
// against 102 with histories of 16,384), of 16,384 leave fewer waves (65).
template <class T, int TILE>
__global__ __launch_bounds__(256) void adjust_kernel(AdjustArgs a) {
  constexpr int V = 16 / sizeof(T);
  constexpr uint32_t kSteps = TILE / (256 * V), kTogether = kSteps < 2 ? kSteps : 2;
  __shared__ uint32_t count[TILE / 2], met[TILE / 32];
  const uint32_t row = blockIdx.y;
  const uint64_t c0 = static_cast<uint64_t>(blockIdx.x) * TILE;
  const uint32_t width = static_cast<uint32_t>(a.n - c0 < TILE ? a.n - c0 : TILE);
  const T* src = static_cast<const T*>(a.scores) + row * a.ld + c0;
  T* dst = static_cast<T*>(a.out) + row * a.out_ld + c0;
  const float* bias = a.bias ? a.bias + row * a.bias_ld + a.first + c0 : nullptr;
  const uint32_t* allow = a.allow ? a.allow + row * a.allow_ld + ((a.first + c0) >> 5) : nullptr;
  Vec<T, V> x[kTogether];
  Vec<float, V> b[kTogether] = {};
  uint32_t on[kTogether];
  auto fetch = [&](uint32_t i0) {
#pragma unroll
    for (uint32_t h = 0; h < kTogether; ++h) {
      const uint32_t i = i0 + h * 256 * V;
      on[h] = allow && i < width ? allow[i >> 5] >> (i & 31) : ~0u;
      if (i + V <= width) {
        x[h] = *reinterpret_cast<const Vec<T, V>*>(src + i);
        if (bias) b[h] = *reinterpret_cast<const Vec<float, V>*>(bias + i);
      }
    }
  };
  const bool history = a.seen && a.seen_n;
  constexpr uint32_t kIds = 8;
  const int32_t* seen = history ? a.seen + row * a.seen_ld : nullptr;
  const uint32_t from = static_cast<uint32_t>(a.first + c0);
  int32_t id[kIds];
  if (history)
#pragma unroll
    for (uint32_t j = 0; j < kIds; ++j) id[j] = threadIdx.x + 256 * j < a.seen_n ? seen[threadIdx.x + 256 * j] : -1;
  fetch(threadIdx.x * V);
  const float r = a.repetition ? a.repetition[row] : 1.0f, f = a.frequency ? a.frequency[row] : 0.0f,
              p = a.presence ? a.presence[row] : 0.0f;
  if (history) {
    for (uint32_t i = threadIdx.x * 4; i < TILE / 2; i += 1024) *reinterpret_cast<uint4*>(&count[i]) = make_uint4(0, 0, 0, 0);
    for (uint32_t i = threadIdx.x; i < TILE / 32; i += 256) met[i] = 0;
    __syncthreads();
    auto meet = [&](int32_t id) {
      const uint32_t at = static_cast<uint32_t>(id) - from;  // ids before the tile and -1 wrap to more than 2^31
      if (at < width) {
        atomicAdd(&count[at >> 1], 1u << (at & 1) * 16);
        atomicOr(&met[at >> 5], 1u << (at & 31));
      }
    };
#pragma unroll
    for (uint32_t j = 0; j < kIds; ++j) meet(id[j]);
    for (uint32_t i = threadIdx.x + 256 * kIds; i < a.seen_n; i += 256) meet(seen[i]);
    __syncthreads();
  }
  auto times = [&](uint32_t i) { return count[i >> 1] >> (i & 1) * 16 & 0xFFFFu; };
  auto penalised = [&](float v, uint32_t times) {
    return ((v > 0.0f ? v / r : v * r) - f * static_cast<float>(times)) - p;
  };
  auto finish = [&](float v, float b, bool on) {
    if (bias) v += b;
    return on ? v : -__builtin_huge_valf();
  };
  for (uint32_t i0 = threadIdx.x * V;;) {
#pragma unroll
    for (uint32_t h = 0; h < kTogether; ++h) {
      const uint32_t i = i0 + h * 256 * V;
      if (i + V <= width) {
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(x[h].v[j]);
        const uint32_t some = history ? met[i >> 5] >> (i & 31) & ((1u << V) - 1) : 0;
        if (some)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (some >> j & 1u) v[j] = penalised(v[j], times(i + j));
#pragma unroll
        for (int j = 0; j < V; ++j) x[h].v[j] = from_f32<T>(finish(v[j], b[h].v[j], on[h] >> j & 1u));
        *reinterpret_cast<Vec<T, V>*>(dst + i) = x[h];
      } else {
        for (uint32_t j = 0; i + j < width; ++j) {
          float v = to_f32(src[i + j]);
          if (history && met[(i + j) >> 5] >> ((i + j) & 31) & 1u) v = penalised(v, times(i + j));
          dst[i + j] = from_f32<T>(finish(v, bias ? bias[i + j] : 0.0f, on[h] >> j & 1u));
        }
      }
    }
    i0 += 256 * V * kTogether;
    if (i0 >= width) break;
    fetch(i0);
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

// A workgroup of 256 threads holds up to kKeys keys and a floor below which nothing can be an answer.  The floor comes from
// counting: the orders of some keys in 256 bins between their least and largest, then the bin that holds the k-th largest in
// 256 finer ones, until few keys are in it: about 1,000 cycles a level, whatever the numbers are, where comparing each of 256
// maxima with each took 4,000 to 6,500.
constexpr uint32_t kKeys = 1024;

struct __attribute__((aligned(16))) Held {
  uint64_t key[kKeys];
  uint32_t bin[256];
  uint32_t least[4], largest[4];  // of each wave
  uint32_t count;
  uint64_t floor;  // keys up to it are no answers, but for those held
};

__device__ inline void begin(Held& h, uint64_t floor = 0) {
  if (threadIdx.x == 0) {
    h.count = 0;
    h.floor = floor;
  }
  __syncthreads();
}

// x of a lane before, for scans over a wave: rows of 16 lanes first, then their last lanes; 0 where there is none
template <int CTRL, int ROWS>
__device__ inline uint32_t before(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xF, false));
}
__device__ inline uint32_t scan_sum(uint32_t x) {  // of the lanes up to this one
  x += before<0x111, 0xF>(x);
  x += before<0x112, 0xF>(x);
  x += before<0x114, 0xF>(x);
  x += before<0x118, 0xF>(x);
  x += before<0x142, 0xA>(x);
  x += before<0x143, 0xC>(x);
  return x;
}
__device__ inline uint32_t of_lane(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}
__device__ inline uint32_t wave_max(uint32_t x) {
  x = max(x, before<0x111, 0xF>(x));
  x = max(x, before<0x112, 0xF>(x));
  x = max(x, before<0x114, 0xF>(x));
  x = max(x, before<0x118, 0xF>(x));
  x = max(x, before<0x142, 0xA>(x));
  x = max(x, before<0x143, 0xC>(x));
  return of_lane(x, 63);
}

// `order`: high words of keys that are all different ones (0: none).  Leaves up to `slack` more than k of them above the
// floor, but for keys of one order.  Ends with a barrier.
template <int M>
__device__ inline void raise_floor(Held& h, const uint32_t (&order)[M], uint32_t k, uint32_t slack) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t largest = 0, inverse = 0;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    largest = max(largest, order[i]);
    inverse = max(inverse, order[i] ? ~order[i] : 0u);
  }
  largest = wave_max(largest);
  inverse = wave_max(inverse);
  if (lane == 0) {
    h.largest[threadIdx.x >> 6] = largest;
    h.least[threadIdx.x >> 6] = ~inverse;
  }
  h.bin[threadIdx.x] = 0;
  __syncthreads();
  uint32_t top = max(max(h.largest[0], h.largest[1]), max(h.largest[2], h.largest[3])),
           base = min(min(h.least[0], h.least[1]), min(h.least[2], h.least[3])), need = k, floor = 0;
  while (base <= top) {  // the same for all threads
    const uint32_t range = top - base, shift = range < 256 ? 0 : 24 - __builtin_clz(range);
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (order[i] >= base && order[i] <= top) atomicAdd(&h.bin[(order[i] - base) >> shift], 1u);
    __syncthreads();
    const uint4 c = reinterpret_cast<const uint4*>(h.bin)[63 - lane];  // lane 0: the highest four
    const uint32_t sum = c.x + c.y + c.z + c.w, reached = scan_sum(sum);
    const uint64_t there = __ballot(reached >= need);
    if (!there) break;  // fewer than k
    const int l = __builtin_ctzll(there);
    uint32_t above = of_lane(reached - sum, l), bin = (63 - l) * 4 + 3, in = of_lane(c.w, l);
    if (above + in < need) above += in, --bin, in = of_lane(c.z, l);
    if (above + in < need) above += in, --bin, in = of_lane(c.y, l);
    if (above + in < need) above += in, --bin, in = of_lane(c.x, l);
    floor = base + (bin << shift);
    need -= above;
    if (shift == 0 || in <= need + slack) break;
    base = floor;
    top = floor + (1u << shift) - 1;
    __syncthreads();
    h.bin[threadIdx.x] = 0;
    __syncthreads();
  }
  if (threadIdx.x == 0 && static_cast<uint64_t>(floor) << 32 > h.floor) h.floor = static_cast<uint64_t>(floor) << 32;
  __syncthreads();
}
__device__ inline uint32_t slack_of(uint32_t k) { return 4 + k / 8; }

// Places the keys whose bits are set, a wave's with one addition to the count; returns the bits of those without room.
template <int N, class Key>
__device__ inline uint32_t place(Held& h, uint32_t pending, Key key) {
  const uint32_t n = __popc(pending), upto = scan_sum(n), all = of_lane(upto, 63);
  if (all == 0) return 0;
  uint32_t at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(&h.count, all);
  at = of_lane(at, 0) + upto - n;
  uint32_t left = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (pending >> i & 1u) {
      if (at < kKeys) h.key[at] = key(i);
      else left |= 1u << i;
      ++at;
    }
  return left;
}

// descending, over the first n (a power of two) keys
__device__ inline void sort_keys(uint64_t* key, uint32_t n) {
  for (uint32_t size = 2; size <= n; size <<= 1)
    for (uint32_t step = size >> 1; step > 0; step >>= 1) {
      for (uint32_t i = threadIdx.x; i < n / 2; i += 256) {
        const uint32_t lo = 2 * i - (i & (step - 1)), hi = lo + step;
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

// Makes room: raises the floor from what is held and drops what does not pass.  Where that leaves more than half (many equal
// values), sorts and keeps the best k.  All threads call it behind a barrier; it ends with one.
__device__ inline void make_room(Held& h, uint32_t k, uint32_t slack) {
  constexpr int M = kKeys / 256;
  const uint32_t held = h.count < kKeys ? h.count : kKeys;
  uint64_t key[M];
  uint32_t order[M];
#pragma unroll
  for (uint32_t i = 0; i < M; ++i) {
    const uint32_t at = i * 256 + threadIdx.x;
    key[i] = at < held ? h.key[at] : 0;
    order[i] = static_cast<uint32_t>(key[i] >> 32);
  }
  raise_floor(h, order, k, slack);
  if (threadIdx.x == 0) h.count = 0;
  __syncthreads();
  const uint64_t floor = h.floor;
  uint32_t kept = 0;
#pragma unroll
  for (uint32_t i = 0; i < M; ++i) kept |= (key[i] && key[i] >= floor ? 1u : 0u) << i;
  place<M>(h, kept, [&](int i) { return key[i]; });
  __syncthreads();
  const uint32_t left = h.count;
  __syncthreads();  // behind it the count may grow again
  if (left <= kKeys / 2) return;
  for (uint32_t i = left + threadIdx.x; i < kKeys; i += 256) h.key[i] = 0;
  __syncthreads();
  sort_keys(h.key, kKeys);
  if (threadIdx.x == 0) {
    h.count = left < k ? left : k;
    if (left >= k) h.floor = h.key[k - 1];
  }
  __syncthreads();
}

// The answers: the best k of what is held, in order.  Ends with a barrier.
__device__ inline void finish(Held& h, uint32_t k) {
  if (h.count > 256) make_room(h, k, min(256 - k, slack_of(k)));
  const uint32_t held = h.count;
  if (held <= 256) {  // each key's place is the number of larger ones
    const uint64_t mine = threadIdx.x < held ? h.key[threadIdx.x] : 0;
    if (threadIdx.x == 0 && held < kKeys) h.key[held] = 0;  // keys are read in twos
    __syncthreads();
    uint32_t place = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < held; i += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&h.key[i]);
      place += (two.x > mine) + (two.y > mine);
    }
    __syncthreads();
    if (threadIdx.x < held) h.key[place] = mine;
  } else {
    for (uint32_t i = held + threadIdx.x; i < kKeys; i += 256) h.key[i] = 0;
    __syncthreads();
    sort_keys(h.key, kKeys);
  }
  __syncthreads();
  if (threadIdx.x == 0) h.count = held < k ? held : k;
  __syncthreads();
}

// Offers each thread's N keys (0: none).  Keys that found no room are offered again behind make_room, which leaves half
// of it, so every turn of the loop places some and it ends.  `first`: raise the floor from them before.
template <int N>
__device__ inline void offer(Held& h, uint32_t k, const uint64_t (&key)[N], bool first) {
  if (first) {
    uint32_t order[N];
#pragma unroll
    for (int i = 0; i < N; ++i) order[i] = static_cast<uint32_t>(key[i] >> 32);
    raise_floor(h, order, k, slack_of(k));
  }
  uint64_t floor = h.floor;
  uint32_t pending = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) pending |= (key[i] > floor ? 1u : 0u) << i;
  for (;;) {
    pending = place<N>(h, pending, [&](int i) { return key[i]; });
    if (!__syncthreads_or(pending != 0)) return;
    make_room(h, k, slack_of(k));
    floor = h.floor;
#pragma unroll
    for (int i = 0; i < N; ++i) pending &= ~((key[i] > floor ? 0u : 1u) << i);
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

// A turn takes 16 values a thread; the next turn's are on their way meanwhile.  The floor is raised from the threads' largest
// values after turns 1, 4, 16, ...: fewer and fewer values then pass it.  Bound by reading: 1024 x 100,003 f32, k = 100, 84 us,
// 4.9 TB/s of the 5.1 that a copy reaches; a short row by the latency of its steps (a slice of 4,096 values 6 us).
template <class T>
__global__ __launch_bounds__(256) void topk_kernel(TopkArgs a, bool to_keys) {
  __shared__ Held h;
  constexpr int V = 16 / sizeof(T), N = 16, L = N / V;  // values of a load, values and loads of a turn
  constexpr float kLowest = -3.402823466e38f;
  const uint32_t row = blockIdx.y, slice = blockIdx.x;
  begin(h);
  const T* src = static_cast<const T*>(a.scores) + row * a.ld;
  const uint64_t per = (a.n + a.slices - 1) / a.slices, c0 = slice * per, c1 = c0 + per < a.n ? c0 + per : a.n;
  Vec<T, V> next[L];
  auto fetch = [&](uint64_t c) {
    if (c + 256 * N <= c1) {
#pragma unroll
      for (int i = 0; i < L; ++i) next[i] = *reinterpret_cast<const Vec<T, V>*>(src + c + i * 256 * V + threadIdx.x * V);
    } else {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const uint64_t at = c + i * 256 * V + threadIdx.x * V;
        if (at + V <= c1) {
          next[i] = *reinterpret_cast<const Vec<T, V>*>(src + at);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) next[i].v[j] = at + j < c1 ? src[at + j] : from_f32<T>(-__builtin_huge_valf());
        }
      }
    }
  };
  if (c0 < c1) fetch(c0);
  float best = -__builtin_huge_valf();
  uint32_t until = 1, turns = 1;
  for (uint64_t c = c0; c < c1; c += 256 * N) {
    float v[N], top[N / 4];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(next[i / V].v[i % V]);
    if (c + 256 * N < c1) fetch(c + 256 * N);
#pragma unroll
    for (int i = 0; i < N / 4; ++i)  // a NaN is no maximum
      top[i] = fmaxf(fmaxf(v[i * 4], v[i * 4 + 1]), fmaxf(v[i * 4 + 2], v[i * 4 + 3]));
    best = fmaxf(best, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    if (--until == 0) {
      const uint32_t order[1] = {best >= kLowest ? static_cast<uint32_t>(key_of(best, 0) >> 32) : 0};
      raise_floor(h, order, a.k, slack_of(a.k));
      until = turns * 3;
      turns *= 4;
    }
    uint64_t floor = h.floor;
    const float low = floor ? key_value(floor) : kLowest;
    auto key = [&](int i) {
      return key_of(v[i], static_cast<uint32_t>(a.first + c + (i / V) * V * 256 + threadIdx.x * V + i % V));
    };
    uint32_t pending = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) pending |= (v[i] >= low ? 1u : 0u) << i;
    for (;;) {  // as offer() does
      if (static_cast<uint32_t>(floor) && pending)  // a floor of its id too
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (pending >> i & 1u && key(i) <= floor) pending &= ~(1u << i);
      pending = place<N>(h, pending, key);
      if (!__syncthreads_or(pending != 0)) break;
      make_room(h, a.k, slack_of(a.k));
      floor = h.floor;
    }
  }
  finish(h, a.k);
  if (to_keys) {
    uint64_t* out = a.keys + (static_cast<uint64_t>(row) * a.key_ld + slice) * a.k;
    for (uint32_t i = threadIdx.x; i < a.k; i += 256) out[i] = i < h.count ? h.key[i] : 0;
  } else {
    write_best(h, a.k, static_cast<T*>(a.values) + static_cast<uint64_t>(row) * a.k,
               a.ids + static_cast<uint64_t>(row) * a.k);
  }
}

// All threads call it behind a barrier.  `key`: of an entry (0: none) and its place in the list.
template <class Entry, class Key>
__device__ inline void offer_list(Held& h, uint32_t k, const Entry* src, uint64_t count, Key key_of_entry) {
  constexpr int N = 8;
  Entry next[N];
  auto fetch = [&](uint64_t c) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t at = c + i * 256 + threadIdx.x;
      next[i] = at < count ? src[at] : 0;
    }
  };
  if (count) fetch(0);
  for (uint64_t c = 0; c < count; c += 256 * N) {
    uint64_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = next[i] ? key_of_entry(next[i], c + i * 256 + threadIdx.x) : 0;
    if (c + 256 * N < count) fetch(c + 256 * N);
    offer(h, k, key, c == 0 && count > k + 64);  // fewer are put in order as fast
  }
}
__device__ inline void offer_list(Held& h, uint32_t k, const uint64_t* keys, uint64_t count) {
  offer_list(h, k, keys, count, [](uint64_t key, uint64_t) { return key; });
}

template <class T>
__global__ __launch_bounds__(256) void merge_kernel(MergeArgs a) {
  __shared__ Held h;
  const uint32_t row = blockIdx.x;
  begin(h);
  offer_list(h, a.k, a.keys + row * a.count, a.count);
  finish(h, a.k);
  write_best(h, a.k, static_cast<T*>(a.values) + static_cast<uint64_t>(row) * a.k,
             a.ids + static_cast<uint64_t>(row) * a.k);
}

// ---------------------------------------------------------------------------------------------- search
// The best k of all records without the score matrix.  A pass scores every stride-th block of 32 records and lists, for
// each query, the keys from its threshold on; the k-th best key of a coarser pass (a lower bound of the k-th best of all
// records) is the next pass's threshold, the coarsest pass stores all its scores, and the last pass is over all records.
// A list whose room ends loses nothing but time: its row is scanned again, alone, where the answers are selected, by one workgroup.
// Lists run full where many records pass that are no answers: a query of scale 0, a threshold or biases too large for the margin
// test (from 1e9 on, below), more equal scores than room.  1024 x 1M x 128, k = 10, takes 0.23 ms; with one query of zeros 8.3, with
// 512 of them 14, with half the records at -1e9 20 (at -1e8 0.23).

// The score as shine_flat_scores and then shine_flat_adjust round it; tb and ab count where the biases are given.
__device__ inline float exact_score(float sum, float qs, float xs, const PassArgs& a, float tb, float ab) {
  float v = (sum * qs) * xs;
  if (a.tbias) v += tb;
  if (a.abias) v += ab;
  return v;
}
__device__ inline float exact_score(float sum, float qs, const PassArgs& a, uint64_t record) {
  return exact_score(sum, qs, a.scales[record], a, a.tbias ? a.tbias[record] : 0.0f, a.abias ? a.abias[record] : 0.0f);
}

__device__ inline uint64_t offered_key(float v, uint64_t record) {
  return v >= -3.402823466e38f ? key_of(v, static_cast<uint32_t>(record)) : 0;
}

// Whether a score reaches the threshold is left to the matrix unit as well.  With the query's scale q and threshold l, the
// record's scale x and bias b,
//   (sum * q) * x + b >= l   <=>   sum + (b / x) (1 / q) - (1 / x) (l / q) >= 0,
// a product of four numbers of the record with four of the query, added to a sum that is already there: kMagic + sum is a
// float (kMagic's), so one 32x32x8 bf16 instruction takes it as its start and leaves the margin in units of the integer
// sum.  Per score that leaves half a maximum to the vector unit, where scaling takes two
// fused multiply-adds (the last pass of 1024 x 1M x 128 fell from 244 to 211 us with it).  A number goes in as two bf16 (2^-17 of it is
// lost), a product as three; the margin is raised by kSlack counts and 2^-13 of its terms, more than this, the roundings of
// the additions and those of the definition come to.  What passes is scored again as the definition rounds.
//
// The terms of a record, and what they meet in a query:
//   u hi          v hi      u = b / x, v = 1 / q
//   u hi          v lo
//   u lo          v hi
//   w hi          y hi      w = 1 / x, y = -l / q
//   w hi          y lo
//   w lo          y hi
//   2^-13 s / x   v hi     s: the sum of the biases' magnitudes, by which their additions round even where they cancel
//   2^-13 w       |y hi|
// The margin still has kMagic in it: the score fails where it is below kMagic, for floats of which some are positive and for
// their bits as integers alike.
constexpr int kSlack = 16;
constexpr float kSumZero = kMagicF + kSlack;  // what a sum of 0 reads as

struct Two {
  __bf16 hi, lo;
  __device__ explicit Two(float x) : hi(static_cast<__bf16>(x)), lo(static_cast<__bf16>(x - static_cast<float>(hi))) {}
};
typedef short v4s __attribute__((ext_vector_type(4)));
struct __attribute__((aligned(16))) Terms {
  __bf16 t[8];
};

// A record for which the margin says nothing always passes (scales and biases whose quotients may overflow), one that is no
// answer never does: its terms are u = +-1e20 alone.  The reciprocals are within 2^-22.
constexpr float kNear = 1e9f, kSure = 1e20f;
// A record of scale 0 is as one of scale 1 if its sums are 0 too: if it has no `codes`.  Each bias on its own may say that it is no
// answer; two finite ones do not, even where their sum b overflows: a large product takes them one after the other.
__device__ inline Terms record_terms(float x, float tb, float ab, bool on, bool codes) {
  const float b = tb + ab, size = fabsf(tb) + fabsf(ab);
  x = x == 0.0f && !codes ? 1.0f : x;
  const bool plain = on && x > 1.0f / kNear && x < kNear && size < kNear;
  const bool none = !on || x != x || !(tb > -__builtin_huge_valf()) || !(ab > -__builtin_huge_valf());
  const float w = plain ? __builtin_amdgcn_rcpf(x) : 0.0f, u = plain ? b * w : none ? -kSure : kSure;
  const Two a(u), c(w);
  return {{a.hi, a.hi, a.lo, c.hi, c.hi, c.lo, static_cast<__bf16>(plain ? 0x1p-13f * (size * w) : 0.0f), static_cast<__bf16>(0x1p-13f * w)}};
}
// Queries for which the margin says nothing (no threshold yet, scales or thresholds whose quotients may overflow) have no
// terms, and a limit that every margin reaches; those that are not there or have no scale one that none does.
__device__ inline bool query_plain(float q, float low) { return q > 1.0f / kNear && q < kNear && fabsf(low) < 1e15f; }
__device__ inline Terms query_terms(float q, float low) {
  if (!query_plain(q, low)) return {{static_cast<__bf16>(0.0f)}};
  const Two v(1.0f / q), y(-low / q);
  return {{v.hi, v.lo, v.hi, y.hi, y.lo, y.hi, v.hi, static_cast<__bf16>(fabsf(static_cast<float>(y.hi)))}};
}
__device__ inline int query_limit(float q, float low, bool there) {
  return !there || q != q ? 0x7FFFFFFF : query_plain(q, low) ? kMagic : -0x7FFFFFFF - 1;
}

// Whether a row has codes other than 0: a scale may be set to 0 with its codes left as they are
__device__ inline bool has_codes(const PassArgs& a, uint64_t record) {
  uint32_t some = 0;
  for (uint32_t c = 0; c < a.pitch; c += 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(a.codes + record * a.pitch + c);
    some |= v.x | v.y | v.z | v.w;
  }
  return some != 0;
}

__device__ inline void write_record_terms(const PassArgs& a, uint64_t block) {  // of 256 records
  const uint64_t r = block * 256 + threadIdx.x;
  if (r >= (a.n + 31) / 32 * 32) return;
  const uint64_t at = min(r, a.n - 1);
  const bool on = r < a.n && (!a.allow || a.allow_ld || (a.allow[r >> 5] >> (r & 31) & 1u));
  const float tb = a.tbias ? a.tbias[at] : 0.0f, ab = a.abias ? a.abias[at] : 0.0f;
  const float x = a.scales[at];
  static_cast<Terms*>(a.record_terms)[r] = record_terms(x, tb, ab, on, x == 0.0f && has_codes(a, at));
}

// Both passes: a wave keeps QT * 32 queries and looks at every fourth block of the workgroup's, in tiles of 32 records x 32
// queries: sum v (0 .. 15) of lane l is of record 8 (v / 4) + 4 (l / 32) + v % 4 and query l % 32.  The next block is fetched while
// this one is scored, with no branch around its loads: behind a branch the loaded registers would be copied, and the copy
// would wait for the loads.
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));

template <int C, int QT>
__device__ inline void load_tile_queries(v4i (&q)[QT][C], const PassArgs& a, uint32_t query0) {
  const uint32_t col = threadIdx.x & 31, half = threadIdx.x >> 5 & 1;
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int8_t* p = a.qcodes + static_cast<uint64_t>(min(query0 + i * 32 + col, a.nq - 1)) * (C * 32) + half * 16;
#pragma unroll
    for (int c = 0; c < C; ++c) q[i][c] = *reinterpret_cast<const v4i*>(p + c * 32);
  }
}
__device__ inline uint32_t records_of(const PassArgs& a, uint64_t word) {
  return static_cast<uint32_t>(min(a.n - word * 32, static_cast<uint64_t>(32)));
}
template <int C>
__device__ inline void load_tile_block(v4i (&x)[C], const PassArgs& a, uint64_t word) {
  const uint32_t col = threadIdx.x & 31, half = threadIdx.x >> 5 & 1;
  const uint32_t at = min(col, records_of(a, word) - 1) * (C * 32) + half * 16;  // behind the last record: the last one
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = *reinterpret_cast<const v4i*>(a.codes + word * (32 * C * 32) + at + c * 32);
}
__device__ inline v16i sums_start() {  // registers of its own, not filled anew for every product
  v16i start;
#pragma unroll
  for (int v = 0; v < 16; ++v) start[v] = kMagic + kSlack;
  asm volatile("" : "+v"(start));
  return start;
}
template <int C>
__device__ inline v16i tile_sums(const v4i (&x)[C], const v4i (&q)[C], const v16i& start) {
  v16i sum = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[0], q[0], start, 0, 0, 0);
#pragma unroll
  for (int c = 1; c < C; ++c) sum = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[c], q[c], sum, 0, 0, 0);
  return sum;
}

// The coarsest pass: a few thousand records of every query; the orders of all their scores are stored, the high words of keys
// whose low ones their places tell.  4,096 records for 1,024 queries take 10 us, their selection 13, the next ones' 6.
template <int KC, int QT>
__global__ __launch_bounds__(256, 2) void sample_kernel(PassArgs a, uint32_t query_blocks, uint64_t per_range) {
  constexpr int C = KC * 2;
  __shared__ float beside[4][3][32];
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 31, half = lane >> 5;
  const Place at = place_of(query_blocks);
  const uint32_t query0 = at.query_block * QT * 32;
  const uint64_t b0 = at.range * per_range, b1 = b0 + per_range < a.blocks ? b0 + per_range : a.blocks;
  if (b0 + wave >= b1) return;
  v4i q[QT][C];
  load_tile_queries<C, QT>(q, a, query0);
  float qs[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) qs[i] = a.qscales[min(query0 + i * 32 + col, a.nq - 1)];
  const v16i start = sums_start();
  for (uint64_t b = b0 + wave; b < b1; b += 4) {
    const uint64_t word = b * a.stride, mine = word * 32 + min(col, records_of(a, word) - 1);
    v4i x[C];
    load_tile_block<C>(x, a, word);
    uint32_t allow[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i)
      allow[i] = a.allow ? a.allow[min(query0 + i * 32 + col, a.nq - 1) * a.allow_ld + word] : ~0u;
    if (half == 0) {
      beside[wave][0][col] = a.scales[mine];
      beside[wave][1][col] = a.tbias ? a.tbias[mine] : 0.0f;
      beside[wave][2][col] = a.abias ? a.abias[mine] : 0.0f;
    }
    wave_sync();
    const uint32_t there = records_of(a, word) == 32 ? ~0u : (1u << records_of(a, word)) - 1;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const uint32_t query = query0 + i * 32 + col;
      const v16i sum = tile_sums<C>(x, q[i], start);
      if (query < a.nq) {
        uint32_t* to = reinterpret_cast<uint32_t*>(a.keys + query * a.cap) + b * 32 + half * 4;
        const uint32_t on = there & allow[i];
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          uint32_t order[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t r = v * 2 + half * 4 + e;
            const float score = exact_score(__int_as_float(sum[v + e]) - kSumZero, qs[i], beside[wave][0][r], a,
                                            beside[wave][1][r], beside[wave][2][r]);
            order[e] = on >> r & 1u ? static_cast<uint32_t>(offered_key(score, 0) >> 32) : 0;
          }
          *reinterpret_cast<uint4*>(to + v * 2) = make_uint4(order[0], order[1], order[2], order[3]);
        }
      }
    }
    wave_sync();
  }
}

// Where a record's 16-byte piece lies in a tile of 32 records in LDS, so that the 8 lanes that one LDS cycle serves meet
// different banks both where they hold neighbouring pieces and where they hold one piece of neighbouring records.
template <int C>
__device__ inline uint32_t tile_piece(uint32_t record, uint32_t piece) {
  return record * (C * 2) + (piece ^ (C % 4 ? record >> 1 & 3 : record & 7));
}

// The other passes: the keys of what reaches the threshold.  A wave lists records and sums in LDS and hands its list on when it
// runs full: only then they are scored (a load of a scale among the tiles would wait for the next block's codes, which are on
// their way) and each query's count is added to once, for additions to one address from all over the GPU are served one after
// another.
//
// Rows of more than 128 codes come by way of LDS: loads of 32 bytes of 32 rows, as the products want them, keep the cache busy
// for about 70 cycles each, four times as long as loads of 1,024 neighbouring bytes (256 x 800k x 200: 109 us a pass, by way of
// LDS 70; without any loads 45).  128 codes: 1024 x 1M x 128, 174 us so and 180 by way of LDS.
//
// 1024 x 1M x 128, last pass: 171 us, 1.6 POP/s of integer products of the 2.1 that a large library product reaches; nothing
// listed 154, and without loads and lists 117.  256 x 200k x 200 with masks, k = 100: 43 us, of which listing 2,900 records a
// query takes 20.
template <int KC, int QT, bool ROWS>
__global__ __launch_bounds__(256, 2) void pass_kernel(PassArgs a, uint32_t query_blocks, uint64_t per_range) {
  constexpr uint32_t kQueries = QT * 32, kList = 512, kFull = kList - 64;  // a turn of the listing adds at most 64 keys
  constexpr int C = KC * 2;
  constexpr bool kTurned = KC > 2;  // the codes come by way of LDS
  struct __attribute__((aligned(16))) Own {  // each wave's
    v4i tile[kTurned ? C * 64 : 1];
    uint2 found[kList];  // record and sum, then the key
    uint32_t query[kList];
    uint32_t count[kQueries], base[kQueries];
    float scale[kQueries];
    uint32_t allow[ROWS ? kQueries : 1];
  };
  __shared__ Own owns[4];
  const uint32_t lane = threadIdx.x & 63, wave = wave_number(), col = lane & 31, half = lane >> 5;
  Own& own = owns[wave];
  const Place at = place_of(query_blocks);
  const uint32_t query0 = at.query_block * kQueries;
  const uint64_t b0 = at.range * per_range, b1 = b0 + per_range < a.blocks ? b0 + per_range : a.blocks, last = b1 - 1;
  if (b0 + wave >= b1) return;
  v4i q[QT][C];
  load_tile_queries<C, QT>(q, a, query0);
  v4s qterms[QT];
  int limit[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const uint32_t query = query0 + i * 32 + col, r = min(query, a.nq - 1);
    qterms[i] = *reinterpret_cast<const v4s*>(&static_cast<const Terms*>(a.query_terms)[r].t[half * 4]);
    limit[i] = query < a.nq ? a.limit[r] : 0x7FFFFFFF;
    if (half == 0) own.scale[i * 32 + col] = a.qscales[r];
  }
  for (uint32_t i = lane; i < kQueries; i += 64) own.count[i] = 0;
  constexpr int MASKS = (kQueries + 63) / 64;  // queries whose mask words a lane fetches
  const uint32_t* allow_row[MASKS];
#pragma unroll
  for (int i = 0; i < MASKS; ++i) allow_row[i] = a.allow + (ROWS ? min(query0 + i * 64 + lane, a.nq - 1) * a.allow_ld : 0);
  const uint32_t* shared_allow = a.allow ? a.allow : reinterpret_cast<const uint32_t*>(a.scales);
  const bool shared = !ROWS && a.allow;
  v4i next[C];
  v4s next_terms;
  uint32_t next_allow[MASKS];
  auto fetch = [&](uint64_t b) {
    const uint64_t word = min(b, last) * a.stride;
    if (kTurned) {
      const uint32_t end = records_of(a, word) * (C * 32) - 16;  // behind the last record: anything
#pragma unroll
      for (uint32_t c = 0; c < C; ++c)
        next[c] = *reinterpret_cast<const v4i*>(a.codes + word * (32 * C * 32) + min(c * 1024 + lane * 16, end));
    } else {
      load_tile_block<C>(next, a, word);
    }
    next_terms = *reinterpret_cast<const v4s*>(&static_cast<const Terms*>(a.record_terms)[word * 32 + col].t[half * 4]);
#pragma unroll
    for (int i = 0; i < MASKS; ++i) next_allow[i] = ROWS ? allow_row[i][word] : i ? 0 : shared_allow[shared ? word : 0];
  };
  uint32_t listed = 0;
  auto hand_on = [&] {
    wave_sync();
    uint32_t place[kList / 64];
#pragma unroll
    for (uint32_t i = 0; i < kList / 64; ++i) {
      place[i] = ~0u;
      if (i * 64 + lane < listed) {
        const uint2 e = own.found[i * 64 + lane];
        const uint32_t mine = own.query[i * 64 + lane];
        const uint64_t key = offered_key(exact_score(__uint_as_float(e.y) - kSumZero, own.scale[mine], a, e.x), e.x);
        own.found[i * 64 + lane] = make_uint2(static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32));
        if (key) place[i] = atomicAdd(&own.count[mine], 1u);
      }
    }
    wave_sync();
    for (uint32_t i = lane; i < kQueries; i += 64) {
      if (own.count[i]) own.base[i] = atomicAdd(&a.count[(query0 + i) * kCountStride], own.count[i]);
      own.count[i] = 0;
    }
    wave_sync();
#pragma unroll
    for (uint32_t i = 0; i < kList / 64; ++i)
      if (place[i] != ~0u) {
        const uint32_t mine = own.query[i * 64 + lane];
        const uint64_t to = static_cast<uint64_t>(own.base[mine]) + place[i];
        const uint2 key = own.found[i * 64 + lane];
        if (to < a.cap) a.keys[(query0 + mine) * a.cap + to] = static_cast<uint64_t>(key.y) << 32 | key.x;
      }
    wave_sync();
    listed = 0;
  };
  const v16i start = sums_start();
  uint32_t to[C], from[C];
#pragma unroll
  for (uint32_t c = 0; c < C; ++c) {
    to[c] = tile_piece<C>((c * 64 + lane) / (C * 2), (c * 64 + lane) % (C * 2));
    from[c] = tile_piece<C>(col, c * 2 + half);
  }
  fetch(b0 + wave);
  for (uint64_t b = b0 + wave; b < b1; b += 4) {
    v4i x[C];
    if (kTurned) {
#pragma unroll
      for (int c = 0; c < C; ++c) own.tile[to[c]] = next[c];
      wave_sync();
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = own.tile[from[c]];
      wave_sync();
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = next[c];
    }
    const v4s terms = next_terms;
    const uint64_t word = b * a.stride;
    const uint32_t there = records_of(a, word);
    const uint32_t live = (there == 32 ? ~0u : (1u << there) - 1) & (shared ? next_allow[0] : ~0u);
    if (ROWS) {
      wave_sync();
#pragma unroll
      for (int i = 0; i < MASKS; ++i)
        if (i * 64 + lane < kQueries) own.allow[i * 64 + lane] = next_allow[i];
      wave_sync();
    }
    fetch(b + 4);
    v16i ahead = tile_sums<C>(x, q[0], start);  // the matrix unit works on the next tile while this one is looked at
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const v16i sum = ahead;
      const v16f margin = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(terms, qterms[i], __builtin_bit_cast(v16f, sum), 0, 0, 0);
      if (i + 1 < QT) ahead = tile_sums<C>(x, q[i + 1 < QT ? i + 1 : 0], start);
      int most = -0x7FFFFFFF - 1;  // as integers, floats' bits keep their order but for the negative ones among themselves
#pragma unroll
      for (int v = 0; v < 16; ++v) most = max(most, __float_as_int(margin[v]));
      if (__any(most >= limit[i])) {
        uint32_t maybe = 0;
#pragma unroll
        for (uint32_t v = 0; v < 16; ++v) maybe |= (__float_as_int(margin[v]) >= limit[i] ? 1u : 0u) << v;
        const uint32_t on = (ROWS ? live & own.allow[i * 32 + col] : live) >> (half * 4);
        maybe &= (on & 15u) | (on >> 4 & 0xF0u) | (on >> 8 & 0xF00u) | (on >> 12 & 0xF000u);
        while (__any(maybe != 0)) {
          const uint32_t v = maybe ? __builtin_ctz(maybe) : 0, r = (v >> 2) * 8 + half * 4 + (v & 3);
          int bits = sum[0];
#pragma unroll
          for (uint32_t e = 1; e < 16; ++e) bits = v == e ? sum[e] : bits;
          const uint64_t who = __ballot(maybe != 0);
          if (maybe) {
            const uint32_t to = listed + __popcll(who & ((1ull << lane) - 1));
            own.found[to] = make_uint2(static_cast<uint32_t>(word * 32 + r), static_cast<uint32_t>(bits));
            own.query[to] = i * 32 + col;
          }
          maybe &= maybe - 1;
          listed += __popcll(who);
          if (listed > kFull) hand_on();
        }
      }
    }
  }
  if (listed) hand_on();
}

// Rows of whole 64-byte steps; a step's four loads are asked for together.
__device__ inline int dot_codes(const int8_t* x, const v4i* q, uint32_t pitch) {
  int sum = 0;
  for (uint32_t c = 0; c < pitch / 64; ++c) {
    v4i v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = reinterpret_cast<const v4i*>(x)[c * 4 + e];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_sdot4(v[e][j], q[c * 4 + e][j], sum, false);
  }
  return sum;
}

__device__ inline uint64_t key_at(const PassArgs& p, uint32_t row, const v4i* query, float qs, uint64_t r) {
  if (r >= p.n || (p.allow && !(p.allow[row * p.allow_ld + (r >> 5)] >> (r & 31) & 1u))) return 0;
  return offered_key(exact_score(static_cast<float>(dot_codes(p.codes + r * p.pitch, query, p.pitch)), qs, p, r), r);
}
__device__ inline void load_query(v4i* query, const PassArgs& p, uint32_t row) {
  if (threadIdx.x < p.pitch / 16)
    query[threadIdx.x] = reinterpret_cast<const v4i*>(p.qcodes + static_cast<uint64_t>(row) * p.pitch)[threadIdx.x];
}

__global__ __launch_bounds__(256) void select_kernel(SelectArgs a) {
  __shared__ Held h;
  __shared__ v4i query[kMaxFusedPitch / 16];
  const PassArgs& p = a.pass;
  const uint32_t row = blockIdx.x;
  if (row >= p.nq) return write_record_terms(p, row - p.nq);
  begin(h);
  const float qs = p.qscales[row];
  const uint64_t listed = a.sample ? p.blocks * 32 : p.count[row * kCountStride];
  if (a.sample)
    offer_list(h, a.k, reinterpret_cast<const uint32_t*>(p.keys + row * p.cap), listed, [&](uint32_t order, uint64_t at) {
      return static_cast<uint64_t>(order) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>((at >> 5) * p.stride * 32 + (at & 31)));
    });
  else
    offer_list(h, a.k, p.keys + row * p.cap, listed < p.cap ? listed : p.cap);
  if (a.extra) offer_list(h, a.k, a.extra + row * a.extra_ld, a.extra_count[row]);
  finish(h, a.k);  // every thread has read the row's count: there is a barrier in between
  if (!a.last) {
    if (threadIdx.x == 0) {
      // a finer pass need not meet the coarser one's records again: where it finds fewer than k, that one's bound stays
      if (h.count == a.k || a.sample) {
        const uint64_t key = h.count == a.k ? h.key[a.k - 1] : 0;
        const float thr = key ? fminf(key_value(key), 3.4028e38f) : -__builtin_huge_valf();  // an infinite one as the largest
        const float low = thr - 0x1p-20f * fabsf(thr);
        static_cast<Terms*>(p.query_terms)[row] = query_terms(qs, low);
        p.limit[row] = query_limit(qs, low, true);
      }
      p.count[row * kCountStride] = 0;
    }
    return;
  }
  if (listed > p.cap) {
    // Keys were lost: all records again, against the floor that the kept ones gave.  The kept ones are met again, so
    // they go; the history's records, which no mask lets through, are offered again.
    load_query(query, p, row);
    const uint64_t floor = h.count == a.k ? h.key[a.k - 1] - 1 : 0;  // the k-th best itself is an answer
    __syncthreads();
    begin(h, floor);
    for (uint64_t r0 = 0; r0 < p.n; r0 += 256) {
      const uint64_t key[1] = {key_at(p, row, query, qs, r0 + threadIdx.x)};
      offer(h, a.k, key, false);
    }
    if (a.extra) offer_list(h, a.k, a.extra + row * a.extra_ld, a.extra_count[row]);
    finish(h, a.k);
  }
  write_best(h, a.k, a.values + static_cast<uint64_t>(row) * a.k, a.ids + static_cast<uint64_t>(row) * a.k);
}

// A search's history is taken out of the passes: seen_mask forbids its records, seen_keys scores them, penalties and all, on
// their own (256 users x 200,000 records with 256 ids each: 12 us, bound by the latency of sorting the ids).
//
// The row's mask without its history: one workgroup per (row, kMaskWords words).
constexpr uint32_t kMaskWords = 4096;
__device__ inline void seen_mask(const SeenArgs& a, uint32_t row, uint64_t w0, uint32_t* mask) {
  const uint32_t width = static_cast<uint32_t>(a.mask_ld - w0 < kMaskWords ? a.mask_ld - w0 : kMaskWords);
  for (uint32_t i = threadIdx.x; i < width; i += 256)
    mask[i] = a.pass.allow ? a.pass.allow[row * a.pass.allow_ld + w0 + i] : 0xFFFFFFFFu;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < a.seen_n; i += 256) {
    const int32_t id = a.seen[row * a.seen_ld + i];
    const int64_t w = static_cast<int64_t>(id >> 5) - static_cast<int64_t>(w0);
    if (id >= 0 && w >= 0 && w < width) atomicAnd(&mask[w], ~(1u << (id & 31)));
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < width; i += 256) a.mask[row * a.mask_ld + w0 + i] = mask[i];
}

// The history's records, each once: the ids sorted in LDS, a run's length its count.
__device__ inline void seen_keys(const SeenArgs& a, uint32_t row, uint32_t* ids, v4i* query, uint32_t& count) {
  const PassArgs& p = a.pass;
  uint32_t n = 2;
  while (n < a.seen_n) n <<= 1;
  for (uint32_t i = threadIdx.x; i < n; i += 256) {
    const int32_t id = i < a.seen_n ? a.seen[row * a.seen_ld + i] : -1;
    ids[i] = id >= 0 && static_cast<uint64_t>(id) < p.n ? static_cast<uint32_t>(id) : 0xFFFFFFFFu;
  }
  if (threadIdx.x < p.pitch / 16)
    query[threadIdx.x] = reinterpret_cast<const v4i*>(p.qcodes + static_cast<uint64_t>(row) * p.pitch)[threadIdx.x];
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  for (uint32_t size = 2; size <= n; size <<= 1)
    for (uint32_t step = size >> 1; step > 0; step >>= 1) {
      for (uint32_t i = threadIdx.x; i < n / 2; i += 256) {
        const uint32_t lo = 2 * step * (i / step) + i % step, hi = lo + step;
        const uint32_t x = ids[lo], y = ids[hi];
        if ((x > y) == ((lo & size) == 0)) {
          ids[lo] = y;
          ids[hi] = x;
        }
      }
      __syncthreads();
    }
  const float qs = p.qscales[row];
  const float rep = a.repetition ? a.repetition[row] : 1.0f, f = a.frequency ? a.frequency[row] : 0.0f,
              pres = a.presence ? a.presence[row] : 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += 256) {
    const uint32_t id = ids[i];
    if (id == 0xFFFFFFFFu || (i > 0 && ids[i - 1] == id)) continue;
    if (p.allow && !(p.allow[row * p.allow_ld + (id >> 5)] >> (id & 31) & 1u)) continue;
    uint32_t lo = i, hi = n;  // the run's end: ids[lo] == id, ids[hi] > id
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (ids[mid] == id) lo = mid; else hi = mid;
    }
    const float times = static_cast<float>(hi - i);
    const float sum = static_cast<float>(dot_codes(p.codes + static_cast<uint64_t>(id) * p.pitch, query, p.pitch));
    float v = (sum * qs) * p.scales[id];
    if (p.tbias) v += p.tbias[id];
    v = ((v > 0.0f ? v / rep : v * rep) - f * times) - pres;
    if (p.abias) v += p.abias[id];
    const uint64_t key = offered_key(v, id);
    if (key) a.extra[row * a.extra_ld + atomicAdd(&count, 1u)] = key;
  }
  __syncthreads();
  if (threadIdx.x == 0) a.extra_count[row] = count;
}

// A row's keys (the first workgroup) and the tiles of its mask.
__global__ __launch_bounds__(256) void seen_kernel(SeenArgs a) {
  static_assert(kMaskWords == kMaxSeen, "one array serves both");
  __shared__ uint32_t words[kMaxSeen];
  __shared__ v4i query[kMaxFusedPitch / 16];
  __shared__ uint32_t count;
  if (blockIdx.x == 0) seen_keys(a, blockIdx.y, words, query, count);
  else seen_mask(a, blockIdx.y, (blockIdx.x - 1ull) * kMaskWords, words);
}

}  // namespace

// The launch's own error.  hipGetLastError would also give, and clear, what an earlier call of the program left behind.
template <class T>
struct As {
  using type = T;
};
template <class... P>
hipError_t launch(void (*kernel)(P...), dim3 grid, hipStream_t s, typename As<P>::type... p) {
  void* args[] = {&p...};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(256), args, 0, s);
}

#define SHINE_BY_ELEM(elem, CALL)                  \
  switch (elem) {                                  \
    case kF32: { using T = float; return CALL; }   \
    case kF16: { using T = __half; return CALL; }  \
    case kBF16: { using T = __bf16; return CALL; } \
    default: return hipErrorInvalidValue;          \
  }

template <class T, int G, int S, int R>
hipError_t quantize_with(const QuantizeArgs& a, uint32_t pitch, hipStream_t s) {
  constexpr uint32_t rows = 256 / G * R;
  const uint64_t groups = std::min<uint64_t>((a.n + rows - 1) / rows, 8192);
  return launch(quantize_kernel<T, G, S, R>, dim3(static_cast<uint32_t>(groups)), s, a, pitch);
}
template <class T>
hipError_t quantize_by_width(const QuantizeArgs& a, hipStream_t s) {
  const uint32_t pitch = code_pitch(a.dim), steps = pitch * sizeof(T) / 16;  // 16-byte steps of a row
  if (steps <= 8) return quantize_with<T, 8, 1, 2>(a, pitch, s);
  if (steps <= 16) return quantize_with<T, 16, 1, 2>(a, pitch, s);
  if (steps <= 32) return quantize_with<T, 32, 1, 2>(a, pitch, s);
  if (steps <= 64) return quantize_with<T, 64, 1, 2>(a, pitch, s);
  if (steps <= 128) return quantize_with<T, 64, 2, 1>(a, pitch, s);
  if (steps <= 256) return quantize_with<T, 64, 4, 1>(a, pitch, s);
  return quantize_with<T, 64, 0, 1>(a, pitch, s);
}

hipError_t launch_quantize(int elem, const QuantizeArgs& a, hipStream_t s) {
  SHINE_BY_ELEM(elem, quantize_by_width<T>(a, s));
}

namespace {
// Ranges of blocks for a streaming launch: about `want` workgroups in all, whole ranges a multiple of 8 (one per XCD).
struct Ranges {
  uint64_t per;
  uint32_t grid;
};
Ranges ranges_of(uint64_t blocks, uint32_t query_blocks, uint32_t want) {
  uint64_t ranges = std::max<uint64_t>(1, want / query_blocks);
  ranges = std::min(ranges, (blocks + 3) / 4);  // four waves take a block each
  const uint64_t per = (blocks + ranges - 1) / ranges;
  const uint64_t whole = ((blocks + per - 1) / per + 7) / 8 * 8;
  return {per, static_cast<uint32_t>(whole * query_blocks)};
}
}  // namespace

template <class T, class E>
hipError_t scores_of_rows(const ScoresArgs& a, hipStream_t s) {
  const Ranges r = ranges_of((a.n + 31) / 32, 1, 1024);
  switch (a.pitch / 64) {
    case 1: return launch(scores_stream_kernel<T, 1, 1, E>, dim3(r.grid), s, a, r.per);
    case 2: return launch(scores_stream_kernel<T, 2, 1, E>, dim3(r.grid), s, a, r.per);
    case 3: return launch(scores_stream_kernel<T, 3, 1, E>, dim3(r.grid), s, a, r.per);
    default: return launch(scores_stream_kernel<T, 4, 1, E>, dim3(r.grid), s, a, r.per);
  }
}

template <class T>
hipError_t scores_of(int elem, const ScoresArgs& a, hipStream_t s) {
  switch (elem) {
    case kF32: return scores_of_rows<T, float>(a, s);
    case kF16: return scores_of_rows<T, __half>(a, s);
    case kBF16: return scores_of_rows<T, __bf16>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_scores_of_rows(int elem, int out_elem, const ScoresArgs& a, hipStream_t s) {
  SHINE_BY_ELEM(out_elem, scores_of<T>(elem, a, s));
}

template <class T, int KC>
hipError_t scores_in_lines_of(const ScoresArgs& a, hipStream_t s) {
  constexpr int QT = 4;
  constexpr uint32_t kLine = 128 / sizeof(T);
  const uint32_t qb = (a.nq + QT * 16 - 1) / (QT * 16);
  const Ranges r = ranges_of((a.n + kLine - 1) / kLine, qb, 512);
  constexpr int P = sizeof(T) == 4 && KC <= 2 ? 2 : 1;
  const uint64_t per = (r.per + 4 * P - 1) / (4 * P) * P;
  return launch(scores_lines_kernel<T, KC, QT, P>, dim3(r.grid), s, a, qb, per);
}

template <class T>
hipError_t scores_of_codes(const ScoresArgs& a, hipStream_t s) {
  // Up to 32 queries: streams (32 x 1M x 128: 45 to 60 us from run to run, in lines 60).  More: lines for rows of 128 codes, and with f32 scores of
  // 256 (1024 x 100,003 x 200: 128 us, in tiles 170); 16-bit scores of wider rows than 128 go in tiles (1024 x 100,000 x 200:
  // 68 us, in lines 119).
  if (a.nq <= 32 && a.pitch <= kStreamPitch) {
    const Ranges r = ranges_of((a.n + 31) / 32, 1, 2048);
    switch (a.pitch / 64) {
      case 1: return launch(scores_stream_kernel<T, 1, 2, void>, dim3(r.grid), s, a, r.per);
      case 2: return launch(scores_stream_kernel<T, 2, 2, void>, dim3(r.grid), s, a, r.per);
      case 3: return launch(scores_stream_kernel<T, 3, 2, void>, dim3(r.grid), s, a, r.per);
      default: return launch(scores_stream_kernel<T, 4, 2, void>, dim3(r.grid), s, a, r.per);
    }
  }
  if (a.nq > 32) {
    if (a.pitch <= 64) return scores_in_lines_of<T, 1>(a, s);
    if (a.pitch <= 128) return scores_in_lines_of<T, 2>(a, s);
    if constexpr (sizeof(T) == 4) {
      if (a.pitch <= 192) return scores_in_lines_of<T, 3>(a, s);
      if (a.pitch <= kStreamPitch) return scores_in_lines_of<T, 4>(a, s);
    }
  }
  // Up to 16 queries: 8 x 100,000 x 768: 21.7 us, in tiles 24.0; 16 x 400,000 x 768: 77.6 and 83.0 (32 in two such tiles a wave:
  // 30.4 us for 100,000, in tiles 25.3).
  if (a.nq <= 16) return launch(scores_few_kernel<T>, dim3(static_cast<uint32_t>((a.n + 127) / 128)), s, a);
  const uint32_t qb = (a.nq + kTileQueries - 1) / kTileQueries, rb = static_cast<uint32_t>((a.n + kTileRecords - 1) / kTileRecords);
  return launch(scores_wide_kernel<T>, dim3((rb + 7) / 8 * 8 * qb), s, a, qb, rb);
}

hipError_t launch_scores(int out_elem, const ScoresArgs& a, hipStream_t s) {
  SHINE_BY_ELEM(out_elem, scores_of_codes<T>(a, s));
}

namespace {
constexpr uint32_t kPassGroups = 512;  // two workgroups a CU

template <int KC, int QT>
hipError_t sample_with(const PassArgs& a, hipStream_t s) {
  const uint32_t qb = (a.nq + QT * 32 - 1) / (QT * 32);
  const Ranges r = ranges_of(a.blocks, qb, kPassGroups);
  return launch(sample_kernel<KC, QT>, dim3(r.grid), s, a, qb, r.per);
}
template <int KC, int QT>
hipError_t pass_with(const PassArgs& a, hipStream_t s) {
  const uint32_t qb = (a.nq + QT * 32 - 1) / (QT * 32);
  const Ranges r = ranges_of(a.blocks, qb, kPassGroups);
  if (a.allow && a.allow_ld) return launch(pass_kernel<KC, QT, true>, dim3(r.grid), s, a, qb, r.per);
  return launch(pass_kernel<KC, QT, false>, dim3(r.grid), s, a, qb, r.per);
}
}  // namespace

hipError_t launch_sample(const PassArgs& a, hipStream_t s) {
  const bool few = a.nq <= 32;
  switch (a.pitch / 64) {
    case 1: return few ? sample_with<1, 1>(a, s) : sample_with<1, 4>(a, s);
    case 2: return few ? sample_with<2, 1>(a, s) : sample_with<2, 4>(a, s);
    case 3: return few ? sample_with<3, 1>(a, s) : sample_with<3, 2>(a, s);
    case 4: return few ? sample_with<4, 1>(a, s) : sample_with<4, 2>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_pass(const PassArgs& a, hipStream_t s) {
  const bool few = a.nq <= 32;  // 32 x 1M x 128: 59 us a call, 63 with room for 128
  switch (a.pitch / 64) {
    case 1: return few ? pass_with<1, 1>(a, s) : pass_with<1, 4>(a, s);
    case 2: return few ? pass_with<2, 1>(a, s) : pass_with<2, 4>(a, s);
    case 3: return few ? pass_with<3, 1>(a, s) : pass_with<3, 2>(a, s);
    case 4: return few ? pass_with<4, 1>(a, s) : pass_with<4, 2>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_select(const SelectArgs& a, hipStream_t s) {
  const uint64_t terms = a.terms ? (a.pass.n + 255) / 256 : 0;
  return launch(select_kernel, dim3(static_cast<uint32_t>(a.pass.nq + terms)), s, a);
}

hipError_t launch_seen(const SeenArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(1 + (a.mask_ld + kMaskWords - 1) / kMaskWords), a.pass.nq);
  return launch(seen_kernel, grid, s, a);
}

hipError_t launch_adjust(int elem, const AdjustArgs& a, hipStream_t s) {
  // Narrow tiles spread a small call over more of the GPU, wide ones read long histories less often (256 x 151,937 f32: 89 us
  // with histories of 8,192, in narrow tiles 128; of 2,048: 61 and 58; 64 x 50,000 with 8,192: 19 and 16).
  const bool wide = a.nq * ((a.n + 8191) / 8192) >= 512;
  const uint64_t tile = wide ? 8192 : 2048;
  const dim3 grid(static_cast<uint32_t>((a.n + tile - 1) / tile), a.nq);
  SHINE_BY_ELEM(elem, launch(wide ? adjust_kernel<T, 8192> : adjust_kernel<T, 2048>, grid, s, a));
}

// Rows are cut where there are too few for the GPU (1 x 1M: 15 us, in one piece 279; 1024 x 20,000: 20.5 either way).
uint32_t topk_slices(uint32_t nq, uint64_t n) {
  const uint64_t want = (1024 + nq - 1) / nq, most = (n + 4095) / 4096;
  const uint64_t s = want < most ? want : most;
  return static_cast<uint32_t>(s ? s : 1);
}

hipError_t launch_topk(int elem, bool keys_only, const TopkArgs& a, hipStream_t s) {
  const bool to_keys = keys_only || a.slices > 1;
  SHINE_BY_ELEM(elem, launch(topk_kernel<T>, dim3(a.slices, a.nq), s, a, to_keys));
}

hipError_t launch_merge(int elem, const MergeArgs& a, hipStream_t s) {
  SHINE_BY_ELEM(elem, launch(merge_kernel<T>, dim3(a.nq), s, a));
}

}  // namespace shine::flat
