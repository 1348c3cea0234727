// norm_kernels.cuh -- the row kernels of the layer / RMS / gated RMS norms, instantiated per I/O type.
//
// With v the row that is normalised (v = s = x + residual, v = x, or v = x silu(z)), n its length:
//   RMS norm:   vh = v rstd,           rstd = (mean(v^2) + eps)^-1/2
//   layer norm: vh = (v - mean) rstd,  rstd = (mean((v - mean)^2) + eps)^-1/2
//   y = vh w + b;   norm before gate: y = vh w silu(z)
// and backwards, with p = dy w (norm before gate: dy w silu(z)):
//   dv = rstd (p - vh mean(p vh) [- mean(p)]),   dw = sum over rows of dy vh,   db = sum over rows of dy.
//
// Every input element is read once and every output element written once. A row's team of threads
// (8 or 16 columns a thread) holds it in registers between its reductions, while the next row's
// asynchronous copies to shared memory are under way, each thread copying what it will read itself. The
// backward forms the row's statistics again (sum v^2 rides along with sum p v) instead of reading saved
// ones. All sums are float32; layer norm subtracts the mean before it squares. Teams walk over the
// rows, so a thread's columns of w (and its running dw, db) stay in registers. The arithmetic goes two
// columns an instruction.
//
// What bounds them: memory, where rows are whole vectors. bf16 rows with a float32 residual, 16384 x 2048:
// forward 67 us (6.0 TB/s of 6.55 that a copy reaches), backward 89 us (6.0); 16384 x 5120 163 (6.2) and 206
// (6.5). bf16 without one: 65536 x 1024 44 us (6.1) and 76 (5.3). The gated norm, 16384 x 4096 bf16: forward
// 64 us (6.3); backward 131 us (5.1), with 2.3 of 4 instructions a cycle from the 16 warps that its registers
// leave an SM. Odd widths take half as many instructions again for the ends of rows: 16384 x 4095 gated 101 us
// (4.0) and 273 (2.5), 65536 x 769 bf16 62 us (3.2) and 117 (2.6). Rows of over 8,192 columns have 64 registers
// a thread (five of the backward bodies for odd widths are given 32) and spill, 76 to 872 bytes forward and 664 to 1,812
// backward: 4096 x 16384 with a float32 residual 141 us (5.7) and 300 (3.6), 4096 x 16383, whose rows are read element by
// element where they do not begin at 16 bytes, 655 (1.2) and 952 (1.1).
//
// Rows that are not 16-byte aligned (odd widths) are still moved 16 bytes at a time: a thread's columns
// begin `phase` columns early, where phase is the row's misalignment, and what the threads at the ends
// of a row then copy of its neighbours is not looked at; only their stores go element by element. The
// phase is one for all rows of a team, because a team's rows lie a multiple of 8 rows apart. A tensor
// whose rows are aligned in another way than the output's is copied in the aligned pieces around a thread's
// columns, and shifted when they are read.
#pragma once

#include <atomic>
#include <type_traits>

#include "norm.cuh"
#include "scan.cuh"

namespace mb200 {

enum { kGateNone = 0, kGateAfterNorm = 1, kGateBeforeNorm = 2 };

constexpr int kCols = 8;           // columns of a vector
constexpr int kPairs = kCols / 2;
__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// A thread's columns: K vectors, the first at column lane * 8 - phase, the others tpr * 8 apart. They are
// the same for all rows. A vector lies inside the row, outside, or (EDGES) across an end of it. Where every
// tensor's rows are aligned and whole vectors wide, EDGES is 0 and the code for the ends is not there
// (16384 x 4096 gated: 64 and 131 us, with it 92 and 251; 131072 x 192: 24 and 37, with it 33 and 73). EDGES is 2
// where some input is to be shifted: 16384 x 2048 bf16 at an odd offset 36 and 69 us, element by element 60 and 104;
// for inputs aligned like the output EDGES 1, without the code for it (16384 x 4095 gated 101 and 273, with it 116 and 312).
template <int K, int EDGES>
struct Columns {
  int first, apart, n;
  bool inside[K];
  __device__ __forceinline__ Columns(int lane, int tpr, int phase, int n) : first(lane * kCols - phase), apart(tpr * kCols), n(n) {
#pragma unroll
    for (int k = 0; k < K; ++k) inside[k] = (*this)[k] >= 0 && (*this)[k] + kCols <= n;
  }
  __device__ __forceinline__ int operator[](int k) const { return first + k * apart; }
  __device__ __forceinline__ bool has(int k, int j) const {
    return EDGES ? (unsigned)((*this)[k] + j) < (unsigned)n : inside[k];
  }
  __device__ __forceinline__ bool meets(int k) const {
    return EDGES ? (*this)[k] < n && (*this)[k] + kCols > 0 : inside[k];
  }
};

__device__ __forceinline__ float& at(float2* x, int j) { return j & 1 ? x[j >> 1].y : x[j >> 1].x; }
__device__ __forceinline__ float at(const float2* x, int j) { return j & 1 ? x[j >> 1].y : x[j >> 1].x; }

// One input tensor: this team's rows of it, and where its pieces lie in a stage of shared memory.
template <typename T, int K, int EDGES>
struct Input {
  using C = Columns<K, EDGES>;
  static constexpr int kPieces = kCols * (int)sizeof(T) / 16;  // 16-byte pieces of a vector
  static constexpr int kUnits = K * kPieces;
  static constexpr int N = kCols / kPieces;            // elements of a piece
  const T* row;  // the next row to copy
  int64_t step;
  bool wide;
  int off;          // elements that a vector begins behind a 16-byte boundary
  uint32_t vector;  // bytes from a vector's pieces to the next one's: a piece more where rows may be shifted

  __device__ __forceinline__ Input(const void* base, int64_t first, int64_t stride, int64_t col0, int64_t team_step,
                                   int phase, uint32_t pitch) {
    row = static_cast<const T*>(base) + first * stride + col0;
    step = team_step * stride;
    const int begin = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (kCols - 1)) - phase;
    wide = (begin & (N - 1)) == 0;
    off = EDGES == 2 ? begin & (N - 1) : 0;
    vector = (kPieces + (EDGES == 2)) * pitch;
  }

  // Copies the row's columns to `slot` (pitch bytes between pieces) and goes on to the next row. `middle`:
  // there are 16 elements of the tensor before the row and 16 behind it, so a vector across its end, and the
  // aligned pieces around one, lie in the tensor too.
  __device__ __forceinline__ void copy(uint32_t slot, uint32_t pitch, const C& c, bool ok, bool middle) {
    if (!EDGES || (middle && wide)) {  // all of a team's threads take one path
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (ok && c.meets(k)) {
#pragma unroll
          for (int u = 0; u < kPieces; ++u) copy_piece(slot + k * vector + u * pitch, row + c[k] + u * N);
        }
    } else if (EDGES == 2 && middle) {  // the aligned pieces that a vector lies in; `read` shifts them
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (c.meets(k)) {
#pragma unroll
          for (int u = 0; u <= kPieces; ++u) copy_piece_l1(slot + k * vector + u * pitch, row + c[k] - off + u * N);
        }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (ok && wide && c.inside[k]) {
#pragma unroll
          for (int u = 0; u < kPieces; ++u) copy_piece(slot + k * vector + u * pitch, row + c[k] + u * N);
        } else if (ok && c.meets(k)) {
          copy_elements(slot + k * vector, pitch, c, k);
        }
      }
    }
    row += step;
  }

  // Vectors outside the row are never copied; where there is no code for ends, their places hold 0 instead.
  static __device__ __forceinline__ void clear(uint32_t slot, uint32_t pitch, const C& c) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (!EDGES && !c.inside[k]) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(slot + (k * kPieces + u) * pitch), "r"(0)
                       : "memory");
      }
  }

  static __device__ __forceinline__ void copy_piece_l1(uint32_t slot, const T* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(src) : "memory");
  }
  // 32-byte vectors by way of L1, where the second piece finds its half of the sector.
  static __device__ __forceinline__ void copy_piece(uint32_t slot, const T* src) {
    if constexpr (kPieces == 1)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(src) : "memory");
    else
      copy_piece_l1(slot, src);
  }

  __device__ __forceinline__ void copy_elements(uint32_t slot, uint32_t pitch, const C& c, int k) {
    constexpr int N = kCols / kPieces;
#pragma unroll 1
    for (int u = 0; u < kPieces; ++u) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < N; ++j) e[j] = c.has(k, u * N + j) ? row[c[k] + u * N + j] : from_f32<T>(0.f);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + u * pitch), "r"(raw.x), "r"(raw.y),
                   "r"(raw.z), "r"(raw.w)
                   : "memory");
    }
  }

  // The copied columns of vector k; those outside the row are 0. (Of a row that there is not, anything: a team
  // without a row stores nothing and adds nothing to dw and db.)
  __device__ __forceinline__ void read(uint32_t slot, uint32_t pitch, const C& c, int k, bool middle, float2* x) const {
    uint32_t w[4 * (kPieces + 1)];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) get_piece(slot + k * vector + u * pitch, w + 4 * u);
    if (EDGES == 2 && off != 0 && middle) {
      constexpr int W = 4 * (kPieces + 1);
      get_piece(slot + k * vector + kPieces * pitch, w + 4 * kPieces);
      const int words = off * (int)sizeof(T) / 4;
#pragma unroll
      for (int i = 0; i + 2 < W; ++i) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i + 1 < W; ++i) w[i] = words & 1 ? w[i + 1] : w[i];
      if (sizeof(T) == 2 && (off & 1)) {
#pragma unroll
        for (int i = 0; i + 1 < W; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
      }
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      if constexpr (kPieces == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = unpack2<T>(w[j]);
      } else {
        x[2 * u] = make_float2(__uint_as_float(w[4 * u]), __uint_as_float(w[4 * u + 1]));
        x[2 * u + 1] = make_float2(__uint_as_float(w[4 * u + 2]), __uint_as_float(w[4 * u + 3]));
      }
    }
    if (EDGES && !c.inside[k]) {
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        if (!c.has(k, j)) at(x, j) = 0.f;
    }
  }
  static __device__ __forceinline__ void get_piece(uint32_t slot, uint32_t* w) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(slot)
                 : "memory");
  }
  __device__ __forceinline__ void read_row(uint32_t slot, uint32_t pitch, const C& c, bool middle,
                                           float2 (&x)[K * kPairs]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) read(slot, pitch, c, k, middle, x + k * kPairs);
  }
};

template <typename T>
__device__ __forceinline__ bool wide_at(const T* row, int phase) {
  return ((reinterpret_cast<uintptr_t>(row) / sizeof(T) ^ phase) & (kCols - 1)) == 0;
}

// Vector k of a row; `wide`: it is aligned there.
template <typename T, int K, int EDGES>
__device__ __forceinline__ void store(T* row, const Columns<K, EDGES>& c, int k, bool ok, bool wide, const float2* x) {
  if (ok && (wide || !EDGES) && c.inside[k]) {
    if constexpr (sizeof(T) == 4)  // a whole sector at once
      asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + c[k]), "f"(x[0].x),
                   "f"(x[0].y), "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y), "f"(x[3].x), "f"(x[3].y)
                   : "memory");
    else
      __stcs(reinterpret_cast<uint4*>(row + c[k]), make_uint4(pack2<T>(x[0]), pack2<T>(x[1]), pack2<T>(x[2]), pack2<T>(x[3])));
  } else if (EDGES && ok && c.meets(k)) {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (c.has(k, j)) row[c[k] + j] = from_f32<T>(at(x, j));
  }
}
template <typename T, int K, int EDGES>
__device__ __forceinline__ void store_row(T* row, const Columns<K, EDGES>& c, bool ok, bool wide, const float2 (&x)[K * kPairs]) {
#pragma unroll
  for (int k = 0; k < K; ++k) store<T, K, EDGES>(row, c, k, ok, wide, x + k * kPairs);
}

// Weight / bias columns as float32; an absent one is `fill`, columns outside are 0.
template <int K, int EDGES>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int64_t col0, const Columns<K, EDGES>& c, float fill,
                                            float2 (&out)[K * kPairs]) {
#pragma unroll
  for (int i = 0; i < K * kCols; ++i) {
    const int64_t col = col0 + c[i / kCols] + i % kCols;
    float v = 0.f;
    if (c.has(i / kCols, i % kCols)) {
      if (w == nullptr)
        v = fill;
      else if (dtype == MB200_F32)
        v = static_cast<const float*>(w)[col];
      else if (dtype == MB200_BF16)
        v = to_f32(static_cast<const __nv_bfloat16*>(w)[col]);
      else
        v = to_f32(static_cast<const __half*>(w)[col]);
    }
    at(out, i) = v;
  }
}

// v -= mean in the columns of the row (those outside stay 0).
template <int K, int EDGES>
__device__ __forceinline__ void centre(float2 (&v)[K * kPairs], const Columns<K, EDGES>& c, float mean) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (c.inside[k]) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[k * kPairs + j] = add2(v[k * kPairs + j], two(-mean));
    } else if (EDGES && c.meets(k)) {
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        if (c.has(k, j)) at(v, k * kCols + j) -= mean;
    }
  }
}

// Sums of one or two values over a row's team; every thread gets them. Up to 32 threads: shuffles inside
// the team. Whole warps: two values are folded into one first (the lower half-warp goes on with the first,
// the upper with the second), and the warps' sums meet in shared memory, where `slot` alternates so that
// one barrier (of the team alone) a sum is enough: a buffer is written again two sums later, after the
// barrier between, which every reader passed.
constexpr unsigned kAllLanes = 0xffffffffu;

template <int S, bool ONE>  // ONE: whole-warp teams have a CTA each
__device__ __forceinline__ void team_sum(float (&v)[S], int tpr, float (*buf)[2][32], int& slot) {
  if (tpr < 32) {  // uniform over the CTA
    for (int off = tpr >> 1; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < S; ++i) v[i] += __shfl_xor_sync(kAllLanes, v[i], off);
    }
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool upper = S == 2 && lane >= 16;
  float s = upper ? v[S - 1] : v[0];
  s += __shfl_xor_sync(kAllLanes, S == 2 ? (upper ? v[0] : v[S - 1]) : s, 16);
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) s += __shfl_xor_sync(kAllLanes, s, off);
  if (tpr > 32) {
    if ((lane & 15) == 0) buf[slot][lane >> 4][warp] = s;  // with one value both halves hold it
    const int warps = tpr >> 5, team = ONE ? 0 : warp / warps;
    if (ONE)
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(tpr) : "memory");
    const float* sums = buf[slot][S == 2 ? lane >> 4 : 0] + team * warps;
    s = 0.f;
    for (int w = lane & 15; w < warps; w += 16) s += sums[w];
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) s += __shfl_xor_sync(kAllLanes, s, off);
    slot ^= 1;
  }
  if (S == 2) {
    const float other = __shfl_xor_sync(kAllLanes, s, 16);
    v[0] = upper ? other : s;
    v[S - 1] = upper ? s : other;
  } else {
    v[0] = s;
  }
}

template <int K>
__device__ __forceinline__ float dot(const float2 (&a)[K], const float2 (&b)[K]) {
  float2 s = two(0.f);
#pragma unroll
  for (int i = 0; i < K; ++i) s = fma2(a[i], b[i], s);
  return s.x + s.y;
}

__device__ __forceinline__ void put4(uint32_t at, float2 a, float2 b) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y) : "memory");
}
__device__ __forceinline__ void get4(uint32_t at, float2& a, float2& b) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a.x), "=f"(a.y), "=f"(b.x), "=f"(b.y) : "r"(at) : "memory");
}

// 1 / (1 + e^-z)
__device__ __forceinline__ float2 sigmoid2_of(float2 z) {
  const float2 t = mul2(z, two(-kLog2e));
  const float2 d = add2(make_float2(ex2(t.x), ex2(t.y)), two(1.f));
  return make_float2(rcp_f(d.x), rcp_f(d.y));
}

// The team of this thread: `lane` of `tpr` threads, its first row, and how far its rows are apart.
struct Team {
  int lane, index;
  int64_t row, step;
};
__device__ __forceinline__ Team find_team(int tpr) {
  const int teams = blockDim.x / tpr;
  Team t;
  t.index = threadIdx.x / tpr;
  t.lane = threadIdx.x - t.index * tpr;
  t.row = (int64_t)blockIdx.x * teams + t.index;
  t.step = (int64_t)gridDim.x * teams;
  return t;
}

// The gated backward keeps a row's sigmoids in shared memory instead of forming them twice (16384 x 4096: 131 us,
// formed twice 148), but not beside rows of over 8,192 columns, for which it has no room.
template <int MAXT>
constexpr bool keep_sigmoids = MAXT <= 640;

template <typename T, typename TR, int GATE>
struct NormTypes {
  static constexpr bool kRes = !std::is_void_v<TR>, kGated = GATE != kGateNone;
  using TS = std::conditional_t<kRes, TR, T>;  // of the rows that are normalised
  // the second (third) input beside x (x and dy): z, the residual, or none
  using TX = std::conditional_t<kGated, T, TS>;
  static constexpr bool kExtra = kRes || kGated;
};

template <typename T, typename TR, int GATE, int K, int MAXT, int EDGES>
__global__ void __launch_bounds__(MAXT, MAXT == 320 ? 2 : 1) norm_fwd_kernel(const NormArgs a, const int tpr, const int nstages) {
  using Types = NormTypes<T, TR, GATE>;
  using TS = typename Types::TS;
  using X = Input<T, K, EDGES>;
  using Extra = Input<typename Types::TX, K, EDGES>;
  constexpr int P = K * kPairs;
  constexpr int more = EDGES == 2 ? K : 0;  // pieces of a row's vectors that shifted rows take besides
  constexpr int kUnits = X::kUnits + more + (Types::kExtra ? Extra::kUnits + more : 0);
  extern __shared__ uint4 stages[];  // [stage][unit][thread]
  __shared__ float buf[2][2][32];
  int slot = 0;
  const Team t = find_team(tpr);
  const int64_t col0 = (int64_t)blockIdx.y * a.n, begin = t.row * a.dim + col0, step = t.step * a.dim;
  const float inv_n = 1.f / (float)a.n;
  T* out = static_cast<T*>(a.out) + begin;
  TS* sum = Types::kRes && a.sum_out != nullptr ? static_cast<TS*>(a.sum_out) + begin : nullptr;
  const int phase = !EDGES || a.no_phase ? 0 : (int)(reinterpret_cast<uintptr_t>(out) / sizeof(T)) & (kCols - 1);
  const bool wide_out = wide_at(out, phase), wide_sum = wide_at(sum, phase);
  const Columns<K, EDGES> c(t.lane, tpr, phase, a.n);
  const void* second = Types::kGated ? a.z : a.residual;
  const int64_t stride2 = Types::kGated ? a.sz : a.sr;
  const uint32_t pitch = blockDim.x * 16, to_extra = (X::kUnits + more) * pitch;
  X x(a.x, t.row, a.sx, col0, t.step, phase, pitch);
  Extra extra(second, t.row, stride2, col0, t.step, phase, pitch);
  const uint32_t mine = smem_of(stages) + threadIdx.x * 16;
  uint32_t read = 0, write = 0;  // stages of the row that is worked on, and of the copies
  const auto in_middle = [&](int64_t row) { return row >= a.margin && row + a.margin < a.rows; };
  const auto copy = [&](int64_t row) {
    const bool ok = row < a.rows, middle = in_middle(row);
    x.copy(mine + write, pitch, c, ok, middle);
    if constexpr (Types::kExtra) extra.copy(mine + write + to_extra, pitch, c, ok, middle);
    asm volatile("cp.async.commit_group;" ::: "memory");
    write = write == (nstages - 1) * kUnits * pitch ? 0 : write + kUnits * pitch;
  };
  for (int k = 0; k < nstages; ++k) {
    X::clear(mine + k * kUnits * pitch, pitch, c);
    if constexpr (Types::kExtra) Extra::clear(mine + k * kUnits * pitch + to_extra, pitch, c);
  }
  for (int k = 0; k + 1 < nstages; ++k) copy(t.row + k * t.step);
  float2 w[P], b[Types::kGated ? 1 : P];
  load_weight<K, EDGES>(a.w, a.w_dtype, col0, c, 1.f, w);
  if constexpr (!Types::kGated) load_weight<K, EDGES>(a.b, a.w_dtype, col0, c, 0.f, b);

  // every thread of a CTA makes the same number of turns (teams past the last row idle)
  for (int64_t row = t.row; row - t.index < a.rows; row += t.step) {
    const bool ok = row < a.rows;
    const uint32_t from = mine + read;
    if (nstages == 1) copy(row);
    if (nstages == 3)
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (nstages > 1) copy(row + (nstages - 1) * t.step);  // into the stage that was read a row ago
    read = read == (nstages - 1) * kUnits * pitch ? 0 : read + kUnits * pitch;
    float2 v[P], g[Types::kExtra ? P : 1];
    x.read_row(from, pitch, c, in_middle(row), v);
    if constexpr (Types::kExtra) extra.read_row(from + to_extra, pitch, c, in_middle(row), g);
    if constexpr (Types::kRes) {
      // the stream is held in its own type; what is normalised is the stream as held
#pragma unroll
      for (int j = 0; j < P; ++j) {
        v[j] = add2(v[j], g[j]);
        if constexpr (sizeof(TS) == 2) v[j] = unpack2<TS>(pack2<TS>(v[j]));
      }
      if (sum != nullptr) {
        store_row<TS, K, EDGES>(sum, c, ok, wide_sum, v);
        sum += step;
      }
    }
    if constexpr (Types::kGated) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        g[j] = mul2(g[j], sigmoid2_of(g[j]));
        if (GATE == kGateBeforeNorm) v[j] = mul2(v[j], g[j]);
      }
    }
    if (!Types::kGated && !a.rms) {
      float2 s2 = two(0.f);
#pragma unroll
      for (int j = 0; j < P; ++j) s2 = add2(s2, v[j]);
      float s[1] = {s2.x + s2.y};
      team_sum<1, true>(s, tpr, buf, slot);
      centre<K, EDGES>(v, c, s[0] * inv_n);
    }
    float q[1] = {dot<P>(v, v)};
    team_sum<1, true>(q, tpr, buf, slot);
    const float rstd = rsqrtf(fmaf(q[0], inv_n, a.eps));
#pragma unroll
    for (int j = 0; j < P; ++j) {
      v[j] = mul2(v[j], two(rstd));
      if constexpr (Types::kGated)
        v[j] = mul2(v[j], w[j]);
      else
        v[j] = fma2(v[j], w[j], b[j]);
      if constexpr (GATE == kGateAfterNorm) v[j] = mul2(v[j], g[j]);
    }
    store_row<T, K, EDGES>(out, c, ok, wide_out, v);
    out += step;
  }
}

template <typename T, typename TR, int GATE, int K, int MAXT, int EDGES>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const NormArgs a, const int tpr, const int nstages) {
  using Types = NormTypes<T, TR, GATE>;
  using TS = typename Types::TS;
  using X = Input<TS, K, EDGES>;
  using Y = Input<T, K, EDGES>;
  using Extra = Input<typename Types::TX, K, EDGES>;
  constexpr bool kGated = Types::kGated, kKeep = keep_sigmoids<MAXT>;
  constexpr int E = K * kCols, P = K * kPairs;
  constexpr int more = EDGES == 2 ? K : 0;
  constexpr int kUnits = X::kUnits + Y::kUnits + 2 * more + (Types::kExtra ? Extra::kUnits + more : 0);
  // [stage][unit][thread], with a gate also the row's sigmoids [4 columns][thread]; behind the last row
  // (teams, n) sums of dw, of db
  extern __shared__ uint4 stages[];
  __shared__ float buf[2][2][32];
  int slot = 0;
  const Team t = find_team(tpr);
  const int64_t col0 = (int64_t)blockIdx.y * a.n, begin = t.row * a.dim + col0, step = t.step * a.dim;
  const float inv_n = 1.f / (float)a.n;
  T* dx = static_cast<T*>(a.dx) + begin;
  TS* dres = Types::kRes && a.dres != nullptr ? static_cast<TS*>(a.dres) + begin : nullptr;
  T* dz = kGated ? static_cast<T*>(a.dz) + begin : nullptr;
  const int phase = !EDGES || a.no_phase ? 0 : (int)(reinterpret_cast<uintptr_t>(dx) / sizeof(T)) & (kCols - 1);
  const bool wide_dx = wide_at(dx, phase), wide_dres = wide_at(dres, phase), wide_dz = wide_at(dz, phase);
  const Columns<K, EDGES> c(t.lane, tpr, phase, a.n);
  const bool extra_given = kGated || a.dsum != nullptr;
  const void* third = kGated ? a.z : a.dsum;
  const int64_t stride3 = kGated ? a.sz : a.dim;
  constexpr uint32_t pitch = MAXT * 16;  // known when the kernel is compiled, unlike blockDim.x
  X x(a.x, t.row, a.sx, col0, t.step, phase, pitch);
  Y y(a.dy, t.row, a.dim, col0, t.step, phase, pitch);
  Extra extra(third, t.row, stride3, col0, t.step, phase, pitch);
  const uint32_t mine = smem_of(stages) + threadIdx.x * 16;
  const uint32_t to_y = (X::kUnits + more) * pitch, to_extra = to_y + (Y::kUnits + more) * pitch;
  const uint32_t sigmoids = mine + nstages * kUnits * pitch;
  uint32_t read = 0, write = 0;  // stages of the row that is worked on, and of the copies
  const auto in_middle = [&](int64_t row) { return row >= a.margin && row + a.margin < a.rows; };
  const auto copy = [&](int64_t row) {
    const bool ok = row < a.rows, middle = in_middle(row);
    x.copy(mine + write, pitch, c, ok, middle);
    y.copy(mine + write + to_y, pitch, c, ok, middle);
    if constexpr (Types::kExtra)
      if (extra_given) extra.copy(mine + write + to_extra, pitch, c, ok, middle);
    asm volatile("cp.async.commit_group;" ::: "memory");
    write = write == (nstages - 1) * kUnits * pitch ? 0 : write + kUnits * pitch;
  };
  for (int k = 0; k < nstages; ++k) {
    X::clear(mine + k * kUnits * pitch, pitch, c);
    Y::clear(mine + k * kUnits * pitch + to_y, pitch, c);
    if constexpr (Types::kExtra) Extra::clear(mine + k * kUnits * pitch + to_extra, pitch, c);
  }
  for (int k = 0; k + 1 < nstages; ++k) copy(t.row + k * t.step);
  float2 w[P], dw[P], db[kGated ? 1 : P];
  load_weight<K, EDGES>(a.w, a.w_dtype, col0, c, 1.f, w);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    dw[j] = two(0.f);
    if constexpr (!kGated) db[j] = two(0.f);
  }

  for (int64_t row = t.row; row - t.index < a.rows; row += t.step) {
    const bool ok = row < a.rows;
    const uint32_t from = mine + read;
    if (nstages == 1) copy(row);
    if (nstages == 3)
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (nstages > 1) copy(row + (nstages - 1) * t.step);  // into the stage that was read a row ago
    read = read == (nstages - 1) * kUnits * pitch ? 0 : read + kUnits * pitch;
    float2 v[P], p[P];
    const bool middle = in_middle(row);
    x.read_row(from, pitch, c, middle, v);
    y.read_row(from + to_y, pitch, c, middle, p);
    if constexpr (kGated) {
      float2 q0 = two(0.f), q1 = two(0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 z[kPairs], sg[kPairs];
        extra.read(from + to_extra, pitch, c, k, middle, z);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) sg[i] = sigmoid2_of(z[i]);
        if (kKeep) {
          put4(sigmoids + 2 * k * pitch, sg[0], sg[1]);
          put4(sigmoids + (2 * k + 1) * pitch, sg[2], sg[3]);
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int j = k * kPairs + i;
          const float2 gate = mul2(z[i], sg[i]);
          float2 pw = mul2(p[j], w[j]);
          if (GATE == kGateBeforeNorm)
            v[j] = mul2(v[j], gate);
          else
            pw = mul2(pw, gate);
          q0 = fma2(v[j], v[j], q0);
          q1 = fma2(pw, v[j], q1);
        }
      }
      float q[2] = {q0.x + q0.y, q1.x + q1.y};
      team_sum<2, false>(q, tpr, buf, slot);
      const float rstd = rsqrtf(fmaf(q[0], inv_n, a.eps));
      const float m = -q[1] * inv_n * rstd * rstd;                     // -vh mean(p vh) / rstd = v m
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 z[kPairs], x0[kPairs], sg[kPairs];  // from shared memory again
        extra.read(from + to_extra, pitch, c, k, middle, z);
        if (kKeep) {
          get4(sigmoids + 2 * k * pitch, sg[0], sg[1]);
          get4(sigmoids + (2 * k + 1) * pitch, sg[2], sg[3]);
        } else {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) sg[i] = sigmoid2_of(z[i]);
        }
        if (GATE == kGateBeforeNorm) x.read(from, pitch, c, k, middle, x0);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int j = k * kPairs + i;
          const float2 gate = mul2(z[i], sg[i]);
          const float2 slope = fma2(gate, fma2(sg[i], two(-1.f), two(1.f)), sg[i]);  // of z sigmoid(z)
          const float2 vh = mul2(v[j], two(rstd));
          const float2 pn = GATE == kGateAfterNorm ? mul2(p[j], gate) : p[j];
          if (ok) dw[j] = fma2(pn, vh, dw[j]);
          const float2 dv = mul2(two(rstd), fma2(v[j], two(m), mul2(pn, w[j])));
          if (GATE == kGateAfterNorm) {
            z[i] = mul2(mul2(p[j], w[j]), mul2(vh, slope));
            v[j] = dv;
          } else {
            z[i] = mul2(dv, mul2(x0[i], slope));
            v[j] = mul2(dv, gate);
          }
        }
        store<T, K, EDGES>(dz, c, k, ok, wide_dz, z);
      }
      dz += step;
    } else {
      float pmean = 0.f;
      if (!a.rms) {
        float2 s2 = two(0.f);
#pragma unroll
        for (int j = 0; j < P; ++j) s2 = add2(s2, v[j]);
        float u[2] = {s2.x + s2.y, dot<P>(p, w)};
        team_sum<2, false>(u, tpr, buf, slot);
        centre<K, EDGES>(v, c, u[0] * inv_n);
        pmean = u[1] * inv_n;
      }
      float2 q1 = two(0.f);
#pragma unroll
      for (int j = 0; j < P; ++j) q1 = fma2(mul2(p[j], w[j]), v[j], q1);
      float q[2] = {dot<P>(v, v), q1.x + q1.y};
      team_sum<2, false>(q, tpr, buf, slot);
      const float rstd = rsqrtf(fmaf(q[0], inv_n, a.eps));
      const float m = -q[1] * inv_n * rstd * rstd;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (ok) {
          dw[j] = fma2(p[j], mul2(v[j], two(rstd)), dw[j]);
          db[j] = add2(db[j], p[j]);
        }
        v[j] = mul2(two(rstd), fma2(v[j], two(m), fma2(p[j], w[j], two(-pmean))));
      }
      if constexpr (Types::kRes) {
        if (extra_given) {
          extra.read_row(from + to_extra, pitch, c, middle, p);
#pragma unroll
          for (int j = 0; j < P; ++j) v[j] = add2(v[j], p[j]);
        }
        if (dres != nullptr) {
          store_row<TS, K, EDGES>(dres, c, ok, wide_dres, v);
          dres += step;
        }
      }
    }
    store_row<T, K, EDGES>(dx, c, ok, wide_dx, v);
    dx += step;
  }
  // This CTA's share of dweight / dbias: one row of `part` per CTA, added up in CTA order by
  // norm_reduce_kernel, so the sums do not depend on the order in which CTAs finish. Of a single CTA they
  // are the gradients.
  if (!a.want_dw && !a.want_db) return;
  const int teams = blockDim.x / tpr;
  const auto put = [&](int col, float sw, float sb) {
    if (gridDim.x == 1) {
      if (a.want_dw) store_grad(a.dw, a.w_dtype, col0 + col, sw);
      if (a.want_db) store_grad(a.db, a.w_dtype, col0 + col, sb);
    } else {
      a.part[(int64_t)blockIdx.x * a.dim + col0 + col] = sw;
      if (a.want_db) a.part[(int64_t)(gridDim.x + blockIdx.x) * a.dim + col0 + col] = sb;
    }
  };
  if (teams > 1) {  // the teams of the CTA first, in order (each has its own phase, so by column)
    float* fold = reinterpret_cast<float*>(stages);
    __syncthreads();  // every thread is done with the copies of its last row
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (c.has(j / kCols, j % kCols)) {
        const int col = c[j / kCols] + j % kCols;
        fold[t.index * a.n + col] = at(dw, j);
        if constexpr (!kGated)
          if (a.want_db) fold[(teams + t.index) * a.n + col] = at(db, j);
      }
    }
    __syncthreads();
    for (int col = threadIdx.x; col < a.n; col += blockDim.x) {
      float sw = 0.f, sb = 0.f;
#pragma unroll 8
      for (int k = 0; k < teams; ++k) {
        sw += fold[k * a.n + col];
        if constexpr (!kGated)
          if (a.want_db) sb += fold[(teams + k) * a.n + col];
      }
      put(col, sw, sb);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (c.has(j / kCols, j % kCols)) {
      float sb = 0.f;
      if constexpr (!kGated) sb = at(db, j);
      put(c[j / kCols] + j % kCols, at(dw, j), sb);
    }
  }
}

// ---- launch: pick the instantiation -----------------------------------------------------------

constexpr int kMostShared = 208 * 1024;  // of an SM's 227 KB, for the copies of the CTAs that it holds

template <typename T, typename TR, int GATE, bool BWD, int K, int MAXT, int EDGES>
cudaError_t norm_run(const NormArgs& a, const NormShape& s, cudaStream_t stream) {
  using Types = NormTypes<T, TR, GATE>;
  constexpr int tensors = (BWD ? 2 : 1) + (Types::kExtra ? 1 : 0);
  constexpr int units = Input<T, K, EDGES>::kUnits + (BWD ? Input<typename Types::TS, K, EDGES>::kUnits : 0) +
                        (Types::kExtra ? Input<typename Types::TX, K, EDGES>::kUnits : 0);
  const int64_t groups = a.dim / a.n;
  dim3 grid((unsigned)s.ctas, (unsigned)groups);
  const auto kernel = BWD ? norm_bwd_kernel<T, TR, GATE, K, MAXT, EDGES> : norm_fwd_kernel<T, TR, GATE, K, MAXT, EDGES>;
  const size_t piece = (size_t)16 * (BWD ? MAXT : s.threads);
  const size_t stage = (units + (EDGES == 2 ? K * tensors : 0)) * piece;
  const size_t sigmoids = BWD && Types::kGated && keep_sigmoids<MAXT> ? K * 2 * piece : 0;
  // Stages of the copies: two rows ahead (16384 x 4096 bf16 with a gate forward 64 us, one row ahead 73), less
  // where the shared memory does not hold them, or where beside two streams that are written more bytes are under
  // way than the memory likes: forward 16384 x 2048 bf16 with a bf16 residual 49 us two rows ahead (80 KB an SM),
  // 44 one row ahead; 16384 x 5120 with a float32 one 176 (61 KB) and 165; but 16384 x 4096 130 (48 KB) and 143.
  // Backward 8192 x 5120 float32 121 and 108, 131072 x 256 bf16 96 and 87, but 16384 x 4096 bf16 174 and 181.
  const size_t row_ahead = (size_t)units * 16 * s.threads * s.resident;
  const bool shallow = Types::kRes && (BWD ? row_ahead >= 56 * 1024 || (K == 1 && s.tpr <= 64) : row_ahead >= 26 * 1024);
  int stages = shallow ? 2 : 3;
  while (stages > 1 && (stages * stage + sigmoids) * s.resident > kMostShared) --stages;
  const int teams = s.threads / s.tpr;
  const size_t fold = BWD && teams > 1 ? sizeof(float) * (a.want_db ? 2 : 1) * teams * (size_t)a.n : 0;
  const size_t smem = stages * stage + sigmoids > fold ? stages * stage + sigmoids : fold;
  // The leave is one number, whatever this call takes: another thread that launches the kernel at another width between
  // these lines and the launch must not lower it.
  static_assert((size_t)(units + (EDGES == 2 ? K * tensors : 0)) * 16 * MAXT +
                        (BWD && Types::kGated && keep_sigmoids<MAXT> ? (size_t)K * 2 * 16 * MAXT : 0) <= kMostShared,
                "a stage of the widest rows");
  if (smem > 40 * 1024) {  // 48 KB, the kernel's own arrays among them, need no leave
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) return e;
  }
  if (!BWD && grid.x > 1) {
    // no more CTAs than the GPU holds at once: what is over would run alone, after the others
    static std::atomic<int> held[kNormMaxThreads / 32 + 1];  // by warps; the shared memory goes by them too
    int per_sm = held[s.threads / 32].load(std::memory_order_relaxed);
    if (per_sm == 0) {
      const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, s.threads, smem);
      if (e != cudaSuccess) return e;
      if (per_sm < 1) per_sm = 1;
      held[s.threads / 32].store(per_sm, std::memory_order_relaxed);
    }
    grid.x = (unsigned)norm_ctas(a, teams, grid.x, most_at_once((int64_t)sm_count() * per_sm, groups));
  }
  kernel<<<grid, s.threads, smem, stream>>>(a, s.tpr, stages);
  return cudaGetLastError();
}

// The most threads of a CTA, and so the registers of a thread: 1024 -> 64, 640 -> 96, 512 -> 128, 384 -> 168.
// A forward CTA of up to 320 threads shares the SM with another (96 registers; 16384 x 4095 gated 168 us alone
// with 128, 112 with another).
template <typename T, typename TR, int GATE, bool BWD, int EDGES>
cudaError_t norm_sized(const NormArgs& a, const NormShape& s, cudaStream_t stream) {
  if (s.k == 1) return norm_run<T, TR, GATE, BWD, 1, 640, EDGES>(a, s, stream);
  if constexpr (!BWD)
    if (s.threads <= 320) return norm_run<T, TR, GATE, BWD, 2, 320, EDGES>(a, s, stream);
  if constexpr (BWD && EDGES)
    if (s.threads <= 384) return norm_run<T, TR, GATE, BWD, 2, 384, EDGES>(a, s, stream);
  if (s.threads <= 512) return norm_run<T, TR, GATE, BWD, 2, 512, EDGES>(a, s, stream);
  return norm_run<T, TR, GATE, BWD, 2, 1024, EDGES != 0>(a, s, stream);  // (rows that wide are not shifted)
}

template <typename T, typename TR, int GATE, bool BWD>
cudaError_t norm_pick(const NormArgs& a, const NormShape& s, cudaStream_t stream) {
  if (!a.edges) return norm_sized<T, TR, GATE, BWD, 0>(a, s, stream);
  return a.shifted ? norm_sized<T, TR, GATE, BWD, 2>(a, s, stream) : norm_sized<T, TR, GATE, BWD, 1>(a, s, stream);
}

template <typename T, bool BWD>
cudaError_t norm_dispatch(const NormArgs& a, const NormShape& s, int res_dtype, cudaStream_t stream) {
  if (a.gate == kGateAfterNorm)
    return norm_pick<T, void, kGateAfterNorm, BWD>(a, s, stream);
  if (a.gate == kGateBeforeNorm)
    return norm_pick<T, void, kGateBeforeNorm, BWD>(a, s, stream);
  if (res_dtype < 0)
    return norm_pick<T, void, kGateNone, BWD>(a, s, stream);
  if (res_dtype == MB200_F32)
    return norm_pick<T, float, kGateNone, BWD>(a, s, stream);
  return norm_pick<T, T, kGateNone, BWD>(a, s, stream);
}

#define MB200_INSTANTIATE_NORM(T)                                                                                 \
  template <>                                                                                                     \
  cudaError_t norm_fwd_of<T>(const NormArgs& a, const NormShape& s, int res_dtype, cudaStream_t stream) {         \
    return norm_dispatch<T, false>(a, s, res_dtype, stream);                                                      \
  }                                                                                                               \
  template <>                                                                                                     \
  cudaError_t norm_bwd_of<T>(const NormArgs& a, const NormShape& s, int res_dtype, cudaStream_t stream) {         \
    return norm_dispatch<T, true>(a, s, res_dtype, stream);                                                       \
  }

}  // namespace mb200
