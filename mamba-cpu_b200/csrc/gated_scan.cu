// gated_scan.cu -- gated linear recurrence over a sequence, forward and backward, and its one-token step.
//
// The steps of a (batch, channel) row are split over lanes: a lane holds 8 consecutive steps, a warp
// a chunk of 256, and one or more warps (of a CTA, or of a small cluster of CTAs) take the chunks of
// a row in turn. Every step is the map h -> a h + b. A lane composes its 8 maps, the lanes of a warp
// join theirs by a shuffle scan, the warps of a row through shared memory (of all CTAs of the
// cluster), and each lane then walks its 8 steps from the state that reaches it. u, the gates and the
// output cross HBM once; nothing per step is kept for the backward but the inputs.
//
// Backward, from the last chunk to the first: with h recomputed inside a chunk from the state that
// entered it (saved by the forward, one float per 256 steps),
//   g_t = dy_t + e_{t+1},  e_t = a_t g_t            the recurrence again, from the other end
//   da = g h_{t-1},  dm = g s_i u,  dla = a da - (a^2 / m) dm
//   du = g m s_i,  d input_gate = g m u s_i (1 - s_i),  d decay_gate = dla A s_r (1 - s_r),  dA = sum dla s_r
//
// What bounds it. A step moves 4 elements forward (2 bytes each in bf16: 8 bytes) and 7 backward, and takes
// 4 special functions forward (two exponentials, a reciprocal and a root; 5 where A < -1: 98 and
// 171 us instead of the 85 and 160 below) and 5 backward, of 34 and 60 instructions in all. 8 x 4096 x 2048 bf16:
// forward 85 us, 6.3 TB/s of 6.55 that a copy reaches, with the special functions 68% busy and 2.9 of 4
// instructions a cycle issued; backward 160 us, 5.9 TB/s, 2.7 instructions a cycle. 1 x 5120 x 65536:
// 456 us (5.9 TB/s) and 817 us (5.75). 4 x 2048 x 2048 float32: 42.6 us (6.3) and 76.5 us (6.1). Packed rows
// whose lengths are no multiple of 8 (3 x 1537 x 1999 fp16): 29 us (2.5) and 46 us (2.8), without ids 19.5 and
// 35: ids and cuts are instructions. A few long rows are bound by the chain of their rounds:
// 64 x 65536 bf16 18 us.
//
// Packed rows: ids (batch, seqlen). A step whose id differs from the one before starts from 0. Steps
// with a negative id are padding: output 0, gradients 0, the state passes through them.
#include <cooperative_groups.h>

#include <type_traits>

#include "gated_scan.cuh"
#include "scan.cuh"

namespace cg = cooperative_groups;

namespace mb200 {

namespace {

constexpr int K = kGatedItems;
constexpr int kPairs = K / 2;
constexpr unsigned kFullMask = 0xffffffffu;

// ---- a lane's 8 steps between memory and registers ------------------------------------------------
//
// Steps travel through shared memory: a warp copies a chunk of every tensor there asynchronously, two
// chunks (one for float32 and packed rows) ahead, in 16-byte pieces, consecutive lanes consecutive pieces. For 16-bit
// types a lane's 8 steps are one piece, its own; for float32 they are two, which two lanes copy, at
// places chosen so that 8 lanes reading one of their pieces each meet all banks. A lane whose steps
// reach past the row's ends, or a tensor whose rows are not aligned like the chunks, is copied element
// by element to the same places.

template <typename T>
constexpr int kVecs = K * (int)sizeof(T) / 16;  // 16-byte pieces of a lane's steps
// Two chunks of 16-bit types ahead: bf16 1 x 6144 x 32768 forward 272 us, backward 496; one ahead 289 and 538
// (8 x 4096 x 2048: 84.6 and 159.6, 86.5 and 157.6). Packed rows, whose ids take shared memory too, one: fp16
// 3 x 1537 x 1999 29.3 and 48.2 us, two ahead 31.5 and 52.
template <typename T, bool IDS>
constexpr int kStages = sizeof(T) == 2 && !IDS ? 3 : 2;
template <typename T, int NT>
constexpr int kTensorBytes = NT * kVecs<T> * 16;  // of a stage, in a CTA of NT threads

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t smem, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Whether wide accesses are aligned on this row: its chunks begin `phase` elements before it.
template <typename T>
__device__ __forceinline__ bool aligned_row(const T* row, int phase) {
  return ((reinterpret_cast<uintptr_t>(row) - phase * sizeof(T)) & (K * sizeof(T) - 1)) == 0;
}

// A thread's places in a tensor's stage: where it copies to (its pieces 512 bytes apart), and its steps.
template <typename T>
struct Places {
  uint32_t to, from[kVecs<T>];
  __device__ __forceinline__ explicit Places(const void* smem) {
    const int lane = threadIdx.x & 31;
    const uint32_t base = smem_address(smem) + (threadIdx.x >> 5) * 32 * kVecs<T> * 16;
    if (kVecs<T> == 1) {
      to = from[0] = base + lane * 16;
    } else {  // piece k lies at k ^ (k / 8 % 2)
      to = base + (lane ^ (lane >> 3 & 1)) * 16;
#pragma unroll
      for (int v = 0; v < kVecs<T>; ++v) from[v] = base + ((lane * 2 + v) ^ (lane >> 2 & 1)) * 16;
    }
  }
};

// A whole chunk of an aligned row, from step c0; `offset`: this tensor's bytes from the first one's.
template <typename T>
__device__ __forceinline__ void copy_chunk(uint32_t to, const T* row, int c0) {
  const T* src = row + (c0 + (int)(threadIdx.x & 31) * (16 / (int)sizeof(T)));
#pragma unroll
  for (int v = 0; v < kVecs<T>; ++v) copy16(to + v * 512, src + v * (512 / (int)sizeof(T)));
}

// A lane's own steps where they may lie outside the row, or the row is not aligned. A piece over an end of
// the row is copied whole all the same where it lies in the tensor (its neighbours' steps are blanked).
template <typename T>
__device__ __forceinline__ void copy_edge(const Places<T>& at, uint32_t offset, const T* row, int t0, int L, bool aligned,
                                          const void* tensor, int64_t elements) {
  if (t0 >= L || t0 + K <= 0) return;
  const T* lo = static_cast<const T*>(tensor);
  const bool whole = aligned && row + t0 >= lo && row + t0 + K <= lo + elements;
#pragma unroll
  for (int v = 0; v < kVecs<T>; ++v) {
    const int t1 = t0 + v * (K / kVecs<T>);
    if (whole) {
      copy16(at.from[v] + offset, row + t1);
    } else {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int j = 0; j < K / kVecs<T>; ++j) e[j] = t1 + j >= 0 && t1 + j < L ? row[t1 + j] : from_f32<T>(0.f);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at.from[v] + offset), "r"(raw.x), "r"(raw.y),
                   "r"(raw.z), "r"(raw.w)
                   : "memory");
    }
  }
}

template <typename T>
__device__ __forceinline__ void unpack(uint4 raw, float2* x) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
    x[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    x[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = unpack2<T>(w[k]);
  }
}

template <typename T>
__device__ __forceinline__ void read_steps(const Places<T>& at, uint32_t offset, float2 (&x)[kPairs]) {
#pragma unroll
  for (int v = 0; v < kVecs<T>; ++v) {
    uint4 raw;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                 : "r"(at.from[v] + offset)
                 : "memory");
    unpack<T>(raw, x + v * (kPairs / kVecs<T>));
  }
}

__device__ __forceinline__ void store_wide(float* p, const float2 (&x)[kPairs]) {  // 32 bytes, a whole sector, at once
  asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0].x), "f"(x[0].y),
               "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y), "f"(x[3].x), "f"(x[3].y)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void store_wide(T* p, const float2 (&x)[kPairs]) {
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(x[0]), pack2<T>(x[1]), pack2<T>(x[2]), pack2<T>(x[3])));
}

// Whether a lane's steps all lie in the row.
__device__ __forceinline__ bool whole_lane(int t0, int L) { return t0 >= 0 && t0 + K <= L; }

template <typename T>
__device__ __forceinline__ void store_edge(T* row, int t0, int L, const float2 (&x)[kPairs]) {
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (t0 + j >= 0 && t0 + j < L) row[t0 + j] = from_f32<T>(j & 1 ? x[j / 2].y : x[j / 2].x);
}

__device__ __forceinline__ float& item(float2 (&x)[kPairs], int j) { return j & 1 ? x[j / 2].y : x[j / 2].x; }

// ---- packed rows -----------------------------------------------------------------------------------

// Bit j of `pad`: step t0 + j is padding or outside the row; of `cut`: it starts a sequence.
struct Marks {
  uint32_t pad, cut;
};

__device__ __forceinline__ uint32_t outside(int t0, int L) {
  const int before = min(max(-t0, 0), K), inside = min(max(L - t0, 0), K);
  return ((1u << before) - 1) | (0xffu & (0xffu << inside));
}

constexpr int kIdSlot = kGatedChunk + 4;  // a chunk's ids, and behind them the id before it

// The warp's ids of the chunk that begins at step c0, padding outside the row.
__device__ __forceinline__ void copy_ids(int32_t* slot, const int32_t* ids, int c0, int L) {
  const int lane = threadIdx.x & 31;
  if (c0 > 0 && c0 + kGatedChunk <= L) {
    const uint32_t to = smem_address(slot) + lane * 4;
    const int32_t* src = ids + (c0 + lane);
#pragma unroll
    for (int j = 0; j < K; ++j) copy4(to + j * 128, src + j * 32);
    if (lane == 0) copy4(to + kGatedChunk * 4, src - 1);
    return;
  }
#pragma unroll 1
  for (int j = 0; j <= K; ++j) {
    const int k = j * 32 + lane;
    if (j == K && lane > 0) break;
    const int t = j == K ? c0 - 1 : c0 + k;
    if (t >= 0 && t < L)
      copy4(smem_address(slot + k), ids + t);
    else
      slot[k] = -1;
  }
}

struct Ids {
  int32_t id[K], prev;
};
__device__ __forceinline__ Ids read_ids(const int32_t* slot) {
  const int lane = threadIdx.x & 31;
  const int4 lo = *reinterpret_cast<const int4*>(slot + lane * K), hi = *reinterpret_cast<const int4*>(slot + lane * K + 4);
  return {{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}, slot[lane > 0 ? lane * K - 1 : kGatedChunk]};
}
// Whether a lane's steps go on with the sequence of the step before them, without padding.
__device__ __forceinline__ bool goes_on(const Ids& x) {
  int32_t differ = 0;
#pragma unroll
  for (int j = 0; j < K; ++j) differ |= x.id[j] ^ x.prev;
  return differ == 0 && x.prev >= 0;
}
__device__ __forceinline__ Marks marks_of(const Ids& x, int t0) {
  Marks m = {0, 0};
  int32_t prev = x.prev;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (x.id[j] < 0) m.pad |= 1u << j;
    if (t0 + j > 0 && x.id[j] >= 0 && x.id[j] != prev) m.cut |= 1u << j;
    prev = x.id[j];
  }
  return m;
}

// ---- joining maps ------------------------------------------------------------------------------------

// Maps h -> A h + B, earlier ones first. Decays are not negative. With CUT an A with its sign bit set has the start
// of a sequence in it: nothing of what came before gets past it, an infinity or a NaN included. (Not an A of 0: that is
// also what fast decays, and products of them, underflow to, and they do pass on an infinity or a NaN. A product with
// a cut in it keeps the sign bit when it underflows.)
constexpr float kCut = -1.f;
__device__ __forceinline__ bool is_cut(float A) { return __float_as_int(A) < 0; }
template <bool CUT>
__device__ __forceinline__ float apply(float A, float B, float h) {
  return CUT && is_cut(A) ? B : fmaf(A, h, B);
}
template <bool CUT>
__device__ __forceinline__ float times(float A, float before) {  // the map A behind the map `before`
  return CUT && is_cut(A) ? A : A * before;
}
template <bool CUT>
__device__ __forceinline__ float decay(float A, float v) {  // of a value, which may be negative
  return CUT && is_cut(A) ? 0.f : A * v;
}

// Inclusive scan of the lanes' maps: from lane 0 up, or (REVERSE) from lane 31 down.
template <bool REVERSE, bool CUT>
__device__ __forceinline__ void scan_maps(int lane, float& A, float& B) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    if (CUT) {
      const float Ap = REVERSE ? __shfl_down_sync(kFullMask, A, off) : __shfl_up_sync(kFullMask, A, off);
      const float Bp = REVERSE ? __shfl_down_sync(kFullMask, B, off) : __shfl_up_sync(kFullMask, B, off);
      if (REVERSE ? lane + off < 32 : lane >= off) {
        B = apply<CUT>(A, B, Bp);
        A = times<CUT>(A, Ap);
      }
    } else if (REVERSE) {  // the shuffle says itself which lanes have a partner
      asm volatile(
          "{\n\t.reg .pred p;\n\t.reg .b32 a, b;\n\t"
          "shfl.sync.down.b32 a|p, %0, %2, 0x1f, 0xffffffff;\n\t"
          "shfl.sync.down.b32 b, %1, %2, 0x1f, 0xffffffff;\n\t"
          "@p fma.rn.f32 %1, %0, b, %1;\n\t@p mul.rn.f32 %0, %0, a;\n\t}"
          : "+f"(A), "+f"(B)
          : "r"(off));
    } else {
      asm volatile(
          "{\n\t.reg .pred p;\n\t.reg .b32 a, b;\n\t"
          "shfl.sync.up.b32 a|p, %0, %2, 0x0, 0xffffffff;\n\t"
          "shfl.sync.up.b32 b, %1, %2, 0x0, 0xffffffff;\n\t"
          "@p fma.rn.f32 %1, %0, b, %1;\n\t@p mul.rn.f32 %0, %0, a;\n\t}"
          : "+f"(A), "+f"(B)
          : "r"(off));
    }
  }
}

// The maps of a row's warps meet here: (A, B) of each warp, two buffers used in turn.
using Exchange = float2[2][kGatedMaxWarps];

// Joins the warps' maps of one round. In: this warp's whole map (A, B) and `carry`, the state that
// enters the round. Out: the state that enters this warp's chunk, and `carry` behind the round. The
// order of the warps is their index, or the reverse of it.
template <bool REVERSE, bool CUT>
__device__ __forceinline__ float join_warps(Exchange& ex, int slot, int self, int warps, int ctas, float A, float B,
                                            float& carry) {
  const int lane = threadIdx.x & 31;
  const int pos = REVERSE ? warps - 1 - self : self;
  if (ctas == 1) {
    if (lane == 0) ex[slot][pos] = make_float2(A, B);
    __syncthreads();
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    if (lane < ctas) *cluster.map_shared_rank(&ex[slot][pos], lane) = make_float2(A, B);
    cluster.sync();
  }
  float2 m = lane < warps ? ex[slot][lane] : make_float2(1.f, 0.f);
  scan_maps<false, CUT>(lane, m.x, m.y);
  const float h = apply<CUT>(m.x, m.y, carry);  // state behind warp `lane`
  const float in = __shfl_sync(kFullMask, h, pos > 0 ? pos - 1 : 0);
  const float mine = pos > 0 ? in : carry;
  carry = __shfl_sync(kFullMask, h, 31);
  return mine;
}

// ---- kernels -----------------------------------------------------------------------------------------

// Which row a warp works on, and which of the row's warps it is.
struct Place {
  int row, b, d, self, phase;
};
__device__ __forceinline__ Place find_place(const GatedScanArgs& a, int warps, int ctas, int3 phase) {
  Place p;
  if (warps == 1) {
    p.row = blockIdx.x;
    p.self = 0;
  } else {
    p.row = blockIdx.x / ctas;
    p.self = (int)(blockIdx.x % ctas) * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5);
  }
  p.b = (unsigned)p.row / (unsigned)a.dim;
  p.d = p.row - p.b * (int)a.dim;
  p.phase = (phase.x + p.b % K * phase.y + p.d % K * phase.z) & (K - 1);
  return p;
}

// x[j] of steps outside the row, or padding, becomes v.
__device__ __forceinline__ void blank(float2 (&x)[kPairs], uint32_t pad, float v) {
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (pad >> j & 1) item(x, j) = v;
}

template <typename T, bool IDS, int NT>
__global__ void __launch_bounds__(NT, NT == 32 ? 21 : 6) gated_fwd_kernel(const GatedScanArgs a, const int row_warps, const int ctas) {
  const int warps = NT == 32 ? 1 : row_warps;
  constexpr int S = kStages<T, IDS>, TB = kTensorBytes<T, NT>;
  extern __shared__ uint4 slots[];  // [stage][u, decay gate, input gate][warp][piece]
  __shared__ Exchange ex;
  __shared__ __align__(16) int32_t id_slots[IDS ? S : 1][NT / 32][IDS ? kIdSlot : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place p = find_place(a, warps, ctas, make_int3(a.phase, a.phase_b, a.phase_d));
  const int L = (int)a.L;
  const T* u = static_cast<const T*>(a.u) + p.b * a.sub + p.d * a.sud;
  const T* r = static_cast<const T*>(a.r) + p.b * a.srb + p.d * a.srd;
  const T* in = static_cast<const T*>(a.i) + p.b * a.sib + p.d * a.sid;
  T* out = static_cast<T*>(a.out) + (int64_t)p.row * L;
  const int32_t* ids = IDS ? a.ids + p.b * a.sqb : nullptr;
  const bool au = aligned_row(u, p.phase), ar = aligned_row(r, p.phase), ai = aligned_row(in, p.phase);
  const bool ao = aligned_row(out, p.phase);
  const float A = checked_decay(a.A[p.d]);
  const bool slow = A >= -1.f;
  if (a.states != nullptr && blockIdx.x == 0 && threadIdx.x == 0)
    *reinterpret_cast<int4*>(a.states) = make_int4(a.phase, a.phase_b, a.phase_d, 0);
  float* states = a.states != nullptr ? a.states + kGatedHeader + (int64_t)p.row * a.chunks : nullptr;
  float carry = a.h0 ? a.h0[p.row] : 0.f;

  const int last = (L + p.phase + kGatedChunk - 1) / kGatedChunk;  // chunks of this row
  const int rounds = (last + warps - 1) / warps;
  const bool aligned = au && ar && ai;
  const Places<T> at(slots);
  const int step = warps * kGatedChunk;
  int begin = p.self * kGatedChunk - p.phase;  // of this round's chunk
  int ahead = begin;                           // of the chunk that is copied next
  uint32_t read = 0, write = 0;                // stages of the two, in bytes
  const auto copy = [&](int round) {
    if (aligned && ahead >= 0 && ahead + kGatedChunk <= L) {
      copy_chunk(at.to + write, u, ahead);
      copy_chunk(at.to + write + TB, r, ahead);
      copy_chunk(at.to + write + 2 * TB, in, ahead);
    } else {
      copy_edge(at, write, u, ahead + lane * K, L, au, a.u, a.u_elements);
      copy_edge(at, write + TB, r, ahead + lane * K, L, ar, a.r, a.r_elements);
      copy_edge(at, write + 2 * TB, in, ahead + lane * K, L, ai, a.i, a.i_elements);
    }
    if (IDS) copy_ids(id_slots[round % S][warp], ids, ahead, L);
    commit_copies();
    ahead += step;
    write = write == (S - 1) * 3 * TB ? 0 : write + 3 * TB;
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) copy(k);
  if (NT > 32 && ctas > 1) cg::this_cluster().sync();  // the other CTAs have started: their shared memory is there

  for (int round = 0; round < rounds; ++round) {
    wait_copies<S - 2>();
    // what other lanes copied has arrived, and all have read the stage that is refilled next
    if (IDS || kVecs<T> > 1) __syncwarp();
    copy(round + S - 1);
    const int t0 = begin + lane * K;
    const bool inner = begin >= 0 && begin + kGatedChunk <= L;
    float2 x[kPairs], gr[kPairs], gi[kPairs], av[kPairs];
    read_steps(at, read, x);
    read_steps(at, read + TB, gr);
    read_steps(at, read + 2 * TB, gi);
    read = read == (S - 1) * 3 * TB ? 0 : read + 3 * TB;
    const auto gates = [&](auto is_slow) {
      constexpr bool kSlow = decltype(is_slow)::value;
      const float2 rate = two(-A);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        float2 q;
        decay2<kSlow>(rate, sigmoid2(gr[k]), av[k], q);
        x[k] = mul2(gated_root2(q, gi[k]), x[k]);
      }
    };
    if (slow)
      gates(std::true_type());
    else
      gates(std::false_type());
    // The recurrence; CUT where the chunk has marks or lies over an end of the row.
    const auto recur = [&](auto is_cut, const Marks mk) {
      constexpr bool CUT = decltype(is_cut)::value;
      const uint32_t pad = mk.pad | (inner ? 0 : outside(t0, L));
      const bool padded = (IDS ? CUT : !inner) && __any_sync(kFullMask, pad != 0);
      if (padded) {
        blank(av, pad, 1.f);
        blank(x, pad, 0.f);
      }
      if (CUT) blank(av, mk.cut, kCut);
      float mA = 1.f, mB = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        mB = apply<CUT>(item(av, j), item(x, j), mB);
        mA = times<CUT>(item(av, j), mA);
      }
      scan_maps<false, CUT>(lane, mA, mB);
      float h = carry;
      if (NT > 32) {
        const float tA = __shfl_sync(kFullMask, mA, 31), tB = __shfl_sync(kFullMask, mB, 31);
        h = join_warps<false, IDS>(ex, round & 1, p.self, warps, ctas, tA, tB, carry);
      }
      const int chunk = round * warps + p.self;
      if (states != nullptr && lane == 0 && chunk < last) states[chunk] = h;
      const float behind = apply<CUT>(mA, mB, h);
      if (NT == 32) carry = __shfl_sync(kFullMask, behind, 31);
      const float before = __shfl_up_sync(kFullMask, behind, 1);
      if (lane > 0) h = before;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        h = apply<CUT>(item(av, j), item(x, j), h);
        item(x, j) = h;
      }
      if (CUT && padded) blank(x, mk.pad, 0.f);
    };
    if constexpr (IDS) {
      const Ids chunk_ids = read_ids(id_slots[round % S][warp]);
      // (a row's warps take one path, on which they meet)
      if (NT == 32 && inner && __all_sync(kFullMask, goes_on(chunk_ids)))
        recur(std::false_type(), Marks{0, 0});
      else
        recur(std::true_type(), marks_of(chunk_ids, t0));
    } else {
      recur(std::false_type(), Marks{0, 0});
    }
    if (ao && whole_lane(t0, L))
      store_wide(out + t0, x);
    else
      store_edge(out, t0, L, x);
    begin += step;
  }
  if (a.last != nullptr && p.self == 0 && lane == 0) a.last[p.row] = carry;
}

template <typename T, bool IDS, int NT>
__global__ void __launch_bounds__(NT, NT == 32 ? 20 : 4) gated_bwd_kernel(const GatedScanArgs a, const int row_warps, const int ctas) {
  const int warps = NT == 32 ? 1 : row_warps;
  constexpr int S = kStages<T, IDS>, TB = kTensorBytes<T, NT>;
  extern __shared__ uint4 slots[];  // [stage][u, decay gate, input gate, dy][warp][piece]
  __shared__ Exchange ex;
  __shared__ float sums[kGatedMaxWarps];
  __shared__ __align__(16) int32_t id_slots[IDS ? S : 1][NT / 32][IDS ? kIdSlot : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 head = a.L > 0 ? *reinterpret_cast<const int4*>(a.states) : make_int4(0, 0, 0, 0);
  const Place p = find_place(a, warps, ctas, make_int3(head.x, head.y, head.z));
  const int L = (int)a.L;
  const T* u = static_cast<const T*>(a.u) + p.b * a.sub + p.d * a.sud;
  const T* r = static_cast<const T*>(a.r) + p.b * a.srb + p.d * a.srd;
  const T* in = static_cast<const T*>(a.i) + p.b * a.sib + p.d * a.sid;
  const T* dy = static_cast<const T*>(a.dout) + (int64_t)p.row * L;
  T* du = static_cast<T*>(a.du) + (int64_t)p.row * L;
  T* dr = static_cast<T*>(a.dr) + (int64_t)p.row * L;
  T* di = static_cast<T*>(a.di) + (int64_t)p.row * L;
  const int32_t* ids = IDS ? a.ids + p.b * a.sqb : nullptr;
  const bool au = aligned_row(u, p.phase), ar = aligned_row(r, p.phase), ai = aligned_row(in, p.phase);
  const bool ay = aligned_row(dy, p.phase);
  const bool ao = aligned_row(du, p.phase) && aligned_row(dr, p.phase) && aligned_row(di, p.phase);
  const float A = checked_decay(a.A[p.d]);
  const bool slow = A >= -1.f;
  float carry = a.dlast ? a.dlast[p.row] : 0.f;  // e behind the last step
  float2 dA = two(0.f);

  const int last = (L + p.phase + kGatedChunk - 1) / kGatedChunk;
  const int rounds = (last + warps - 1) / warps;
  // turn 0 is the row's last round
  const bool aligned = au && ar && ai && ay;
  const Places<T> at(slots);
  const int step = warps * kGatedChunk;
  int chunk = (rounds - 1) * warps + p.self;
  int begin = chunk * kGatedChunk - p.phase;  // of this turn's chunk
  int ahead = begin;                          // of the chunk that is copied next
  uint32_t read = 0, write = 0;               // stages of the two, in bytes
  const auto copy = [&](int turn) {
    if (aligned && ahead >= 0 && ahead + kGatedChunk <= L) {
      copy_chunk(at.to + write, u, ahead);
      copy_chunk(at.to + write + TB, r, ahead);
      copy_chunk(at.to + write + 2 * TB, in, ahead);
      copy_chunk(at.to + write + 3 * TB, dy, ahead);
    } else {
      copy_edge(at, write, u, ahead + lane * K, L, au, a.u, a.u_elements);
      copy_edge(at, write + TB, r, ahead + lane * K, L, ar, a.r, a.r_elements);
      copy_edge(at, write + 2 * TB, in, ahead + lane * K, L, ai, a.i, a.i_elements);
      copy_edge(at, write + 3 * TB, dy, ahead + lane * K, L, ay, a.dout, a.batch * a.dim * a.L);
    }
    if (IDS) copy_ids(id_slots[turn % S][warp], ids, ahead, L);
    commit_copies();
    ahead -= step;
    write = write == (S - 1) * 4 * TB ? 0 : write + 4 * TB;
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) copy(k);
  if (NT > 32 && ctas > 1) cg::this_cluster().sync();  // the other CTAs have started: their shared memory is there
  const float* states = a.states + kGatedHeader + (int64_t)p.row * a.chunks;  // the state that entered each chunk
  float next = chunk >= 0 && chunk < last ? states[chunk] : 0.f;

  for (int turn = 0; turn < rounds; ++turn) {
    wait_copies<S - 2>();
    if (IDS || kVecs<T> > 1) __syncwarp();
    copy(turn + S - 1);
    const int t0 = begin + lane * K;
    const bool inner = begin >= 0 && begin + kGatedChunk <= L;
    float h = next;
    chunk -= warps;
    next = chunk >= 0 && chunk < last ? states[chunk] : 0.f;
    float2 x[kPairs], sr[kPairs], si[kPairs], g[kPairs], av[kPairs], m[kPairs], inv[kPairs], hp[kPairs];
    read_steps(at, read, x);
    read_steps(at, read + TB, sr);
    read_steps(at, read + 2 * TB, si);
    const auto gates = [&](auto is_slow) {
      constexpr bool kSlow = decltype(is_slow)::value;
      const float2 rate = two(-A);
      // The root's slope, infinite at q = 0, is 0 in a channel whose A is 0. In others q is 0 where a gate
      // is shut, and s_r times any finite slope is 0 too: a number as small as gated_root2's is added.
      const float2 tiny = two(A == 0.f ? __int_as_float(0x7f800000) : 1e-37f);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        float2 q;
        sr[k] = sigmoid2(sr[k]);
        si[k] = sigmoid2(si[k]);
        decay2<kSlow>(rate, sr[k], av[k], q);
        const float2 root = add2(q, tiny);
        inv[k] = make_float2(rsqrt_f(root.x), rsqrt_f(root.y));
        m[k] = mul2(q, inv[k]);
        hp[k] = mul2(mul2(m[k], si[k]), x[k]);
        inv[k] = mul2(mul2(av[k], av[k]), inv[k]);  // -dm / dla = a^2 / m
      }
    };
    if (slow)
      gates(std::true_type());
    else
      gates(std::false_type());
    read_steps(at, read + 3 * TB, g);
    const uint32_t mine = read;
    read = read == (S - 1) * 4 * TB ? 0 : read + 4 * TB;
    // The recurrences and the gradients; CUT where the chunk has marks or lies over an end of the row.
    const auto recur = [&](auto is_cut, const Marks mk) {
      constexpr bool CUT = decltype(is_cut)::value;
      const uint32_t pad = mk.pad | (inner ? 0 : outside(t0, L));
      const bool padded = (IDS ? CUT : !inner) && __any_sync(kFullMask, pad != 0);
      if (padded) {
        blank(av, pad, 1.f);
        blank(hp, pad, 0.f);
        blank(g, pad, 0.f);
      }
      if (CUT) blank(av, mk.cut, kCut);
      // the chunk's states again: hp[j] becomes the state before step j
      float mA = 1.f, mB = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        mB = apply<CUT>(item(av, j), item(hp, j), mB);
        mA = times<CUT>(item(av, j), mA);
      }
      const float whole = mA;
      scan_maps<false, CUT>(lane, mA, mB);
      const float before = __shfl_up_sync(kFullMask, apply<CUT>(mA, mB, h), 1);
      if (lane > 0) h = before;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const float after = apply<CUT>(item(av, j), item(hp, j), h);
        item(hp, j) = h;
        h = after;
      }
      // e from the end: the map of a step is e -> a (dy + e)
      mA = whole, mB = 0.f;
#pragma unroll
      for (int j = K - 1; j >= 0; --j) mB = decay<CUT>(item(av, j), item(g, j) + mB);
      scan_maps<true, CUT>(lane, mA, mB);
      float e = carry;
      if (NT > 32) {
        const float tA = __shfl_sync(kFullMask, mA, 0), tB = __shfl_sync(kFullMask, mB, 0);
        e = join_warps<true, IDS>(ex, turn & 1, p.self, warps, ctas, tA, tB, carry);
      }
      const float ahead_e = apply<CUT>(mA, mB, e);
      if (NT == 32) carry = __shfl_sync(kFullMask, ahead_e, 0);
      const float later = __shfl_down_sync(kFullMask, ahead_e, 1);
      if (lane < 31) e = later;
#pragma unroll
      for (int j = K - 1; j >= 0; --j) {  // g = dy + e; av becomes a g
        item(g, j) += e;
        e = decay<CUT>(item(av, j), item(g, j));
        item(av, j) = e;
        if (CUT && (mk.cut >> j & 1)) item(hp, j) = 0.f;
      }
      read_steps(at, mine, x);  // u once more: eight registers less in between
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const float2 gs = mul2(g[k], si[k]);  // dm / u
        const float2 gu = mul2(gs, x[k]);
        const float2 du2 = mul2(gs, m[k]);
        float2 ds = fma2(mul2(inv[k], gu), two(-1.f), mul2(av[k], hp[k]));  // dla
        ds = mul2(ds, sr[k]);
        x[k] = du2;
        si[k] = mul2(mul2(gu, m[k]), fma2(si[k], two(-1.f), two(1.f)));
        sr[k] = mul2(mul2(ds, two(A)), fma2(sr[k], two(-1.f), two(1.f)));
        hp[k] = ds;
      }
      if (padded) {
        blank(x, pad, 0.f);
        blank(si, pad, 0.f);
        blank(sr, pad, 0.f);
        blank(hp, pad, 0.f);
      }
#pragma unroll
      for (int k = 0; k < kPairs; ++k) dA = add2(dA, hp[k]);
    };
    if constexpr (IDS) {
      const Ids chunk_ids = read_ids(id_slots[turn % S][warp]);
      // (a row's warps take one path, on which they meet)
      if (NT == 32 && inner && __all_sync(kFullMask, goes_on(chunk_ids)))
        recur(std::false_type(), Marks{0, 0});
      else
        recur(std::true_type(), marks_of(chunk_ids, t0));
    } else {
      recur(std::false_type(), Marks{0, 0});
    }
    if (ao && whole_lane(t0, L)) {
      store_wide(du + t0, x);
      store_wide(dr + t0, sr);
      store_wide(di + t0, si);
    } else {
      store_edge(du, t0, L, x);
      store_edge(dr, t0, L, sr);
      store_edge(di, t0, L, si);
    }
    begin -= step;
  }
  float sum = dA.x + dA.y;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
  if (NT > 32) {
    if (ctas == 1) {
      if (lane == 0) sums[p.self] = sum;
      __syncthreads();
    } else {
      cg::cluster_group cluster = cg::this_cluster();
      if (lane == 0) *cluster.map_shared_rank(&sums[p.self], 0) = sum;
      cluster.sync();
    }
    if (p.self != 0) return;
    sum = lane < warps ? sums[lane] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
  }
  if (lane == 0) {
    a.part[p.row] = sum;
    if (a.dh0 != nullptr) a.dh0[p.row] = carry;
  }
}

// dA[d] = sum over the batch, in order. (4 bytes a row of the scan: 4.5 us from cold caches at 4 x 4096 rows.)
__global__ void gated_reduce_kernel(const float* part, int64_t batch, int64_t dim, float* dA) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= dim) return;
  float s = 0.f;
  for (int64_t b = 0; b < batch; ++b) s += part[b * dim + d];
  dA[d] = s;
}

// One step of every channel: 10 bytes read and 6 written an element with a float32 state and bf16 inputs, and
// no chain, so the launch bounds a few rows and memory the rest. 4 elements a thread where addresses allow it:
// 256 x 5120 4.6 us (launch included; 8.7 one at a time), 4096 x 5120 50.0 us, 6.7 TB/s (105).
template <typename T, typename TS, int V>
__global__ void __launch_bounds__(128) gated_step_kernel(const GatedStepArgs a) {
  const int64_t per_row = a.dim / V;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.batch * per_row) return;
  const int64_t b = i / per_row, d = (i % per_row) * V;
  float u[V], r[V], g[V], A[V], h[V];
  load_cached<T, V>(static_cast<const T*>(a.u) + b * a.su + d, u);
  load_cached<T, V>(static_cast<const T*>(a.r) + b * a.sr + d, r);
  load_cached<T, V>(static_cast<const T*>(a.i) + b * a.si + d, g);
  load_cached<float, V>(a.A + d, A);
#pragma unroll
  for (int j = 0; j < V; ++j) A[j] = checked_decay(A[j]);
  {
    // not the read-only path: new_state may be state itself
    using R = RowVec<TS, V>;
    const auto* p = reinterpret_cast<const typename R::V*>(static_cast<const TS*>(a.state) + b * a.ss + d);
#pragma unroll
    for (int v = 0; v < R::kNV; ++v) {
      const typename R::V raw = p[v];
      const TS* e = reinterpret_cast<const TS*>(&raw);
#pragma unroll
      for (int j = 0; j < R::kEPV; ++j) h[v * R::kEPV + j] = to_f32<TS>(e[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const int k = j + 1 < V ? j + 1 : j;
    float2 aj, q;
    decay2<false>(make_float2(-A[j], -A[k]), sigmoid2(make_float2(r[j], r[k])), aj, q);
    const float2 in = mul2(gated_root2(q, make_float2(g[j], g[k])), make_float2(u[j], u[k]));
    const float2 nh = fma2(aj, make_float2(h[j], h[k]), in);
    h[j] = nh.x;
    if (k > j) h[k] = nh.y;
  }
  store_stream<TS, V>(static_cast<TS*>(a.new_state) + b * a.sn + d, h);
  store_stream<T, V>(static_cast<T*>(a.out) + b * a.dim + d, h);
}

// Warps of a row, four to a CTA, the CTAs of a row in a cluster: as many as it takes to give the GPU 14 warps
// an SM, but no more than the row has chunks, and clusters only for rows of 16 chunks and more. Forward and
// backward of bf16 rows of 8,192 steps, in us, by warps a row:
//   rows    1           2           4           8           16          32
//     64    15.5 23.8   12.8 17.0    7.6  9.9    7.3  9.2    5.1  6.9    4.6  6.3
//    160    15.6 23.9   12.9 17.0    8.4 11.4    8.3 10.9    6.5 14.6    8.7 16.3
//    512    17.1 25.9   16.1 22.1   12.6 18.7   17.7 26.2   17.7 33.7   21.5 44.9
//   1024    20.4 32.6   21.2 31.5   20.9 31.0   27.8 48.8   30.7 61.5   40.2 84.1
//   1536    25.0 41.3   27.6 46.4   26.3 43.8   37.6 69.4   44.1 86.3   58.8 122
// and of 64 rows of 2,048 steps (8 chunks): 3.4 4.3 at 4, 3.5 4.8 at 8.
//
// A row that is one warp's has a CTA of one warp: starting a CTA takes about as long as three chunks, and
// four warps that start (and end) together leave more of that uncovered than four that do so one by one.
void row_split(const GatedScanArgs& a, int* warps, int* ctas) {
  const int64_t rows = a.batch * a.dim, chunks = (a.L + kGatedChunk - 1) / kGatedChunk;
  int64_t want = (int64_t)sm_count() * 14 / rows;
  if (want > chunks) want = chunks;
  if (chunks < 16 && want > 4) want = 4;
  int w = 1;
  while (w * 2 <= want && w < kGatedMaxWarps) w *= 2;
  *ctas = w > 4 ? w / 4 : 1;
  *warps = w;
}

constexpr int kLongRow = 32;  // chunks
// One-warp forward CTAs without ids that an SM holds (32 is its most; float32 rows take 7.5 KB of shared memory each),
// and the most rows an SM of which a second wave is small enough to be evened out.
template <typename T>
constexpr int kMostCtas = sizeof(T) == 4 ? 29 : 32;
constexpr int kMostEvened = 45;
constexpr int kSmSharedBytes = 228 * 1024, kCtaSharedBytes = 1024;  // of an SM; taken by a CTA besides its request

template <typename T, bool IDS, int TENSORS, int NT, typename F>
cudaError_t launch_rows(F kernel, const GatedScanArgs& a, int warps, int ctas, cudaStream_t stream) {
  const int64_t rows = a.batch * a.dim;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(32 * warps / ctas);
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.dynamicSmemBytes = kStages<T, IDS> * TENSORS * kTensorBytes<T, NT>;  // 32 KB at most
  if (TENSORS == 3 && !IDS && warps == 1 && a.chunks >= kLongRow) {
    // Long rows in a full and a nearly empty wave: fewer at a time (by asking for more shared memory than is used), so
    // that the second wave is not left to a few warps. Forward of 1 x 5120 x 65536 bf16, 35 rows an SM: 492 us at 32 at a
    // time, 461 at 20. Rows of 16,384 steps, us as many at a time as fit and evened out, by rows an SM:
    //   bf16     33  119 119   35  128 121   38  138 134   40  140 140   42  140 142   44  148 144   46  150 154   56  175 183
    //   float32  30  191 185   33  220 203   35  257 210   38  259 222   40  267 250   44  279 271   46  283 283   48  285 289
    // Packed rows, which registers hold to 25, lose (bf16 1 x 5120 x 65536 568 and 578, float32 1 x 5120 x 32768 431 and
    // 446), and so do rows of 2,048 steps (8 x 4096 x 2048 bf16 85 us at 32 at a time, 91 at 20). Registers (85 to 92 a
    // thread) hold the backward to 20 rows an SM anyway.
    const int64_t per_sm = (rows + sm_count() - 1) / sm_count(), fewer = (per_sm + 1) / 2 + 2;
    if (per_sm > kMostCtas<T> && per_sm <= kMostEvened) {
      const size_t share = ((size_t)kSmSharedBytes / fewer - kCtaSharedBytes) / 128 * 128;
      if (share > cfg.dynamicSmemBytes) cfg.dynamicSmemBytes = share;
    }
  }
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, static_cast<int>(warps), static_cast<int>(ctas));
}

template <typename T, bool IDS>
cudaError_t fwd_ids(const GatedScanArgs& a, cudaStream_t stream) {
  int warps, ctas;
  row_split(a, &warps, &ctas);
  return warps == 1 ? launch_rows<T, IDS, 3, 32>(gated_fwd_kernel<T, IDS, 32>, a, warps, ctas, stream)
                    : launch_rows<T, IDS, 3, 128>(gated_fwd_kernel<T, IDS, 128>, a, warps, ctas, stream);
}

template <typename T, bool IDS>
cudaError_t bwd_ids(const GatedScanArgs& a, cudaStream_t stream) {
  int warps, ctas;
  row_split(a, &warps, &ctas);
  return warps == 1 ? launch_rows<T, IDS, 4, 32>(gated_bwd_kernel<T, IDS, 32>, a, warps, ctas, stream)
                    : launch_rows<T, IDS, 4, 128>(gated_bwd_kernel<T, IDS, 128>, a, warps, ctas, stream);
}

template <typename T>
cudaError_t fwd_of(const GatedScanArgs& a, cudaStream_t stream) {
  return a.ids ? fwd_ids<T, true>(a, stream) : fwd_ids<T, false>(a, stream);
}

template <typename T>
cudaError_t bwd_of(const GatedScanArgs& a, cudaStream_t stream) {
  return a.ids ? bwd_ids<T, true>(a, stream) : bwd_ids<T, false>(a, stream);
}

template <typename T, typename TS>
cudaError_t step_of(const GatedStepArgs& a, cudaStream_t stream) {
  constexpr int V = 4;
  const int64_t n = a.batch * a.dim / (a.vec ? V : 1);
  const unsigned grid = (unsigned)((n + 127) / 128);
  if (a.vec)
    gated_step_kernel<T, TS, V><<<grid, 128, 0, stream>>>(a);
  else
    gated_step_kernel<T, TS, 1><<<grid, 128, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gated_scan_fwd(const GatedScanArgs& a, int dtype, cudaStream_t stream) {
  if (a.batch * a.dim == 0) return cudaSuccess;
  note_launches(1);
  switch (dtype) {
    case MB200_F32: return fwd_of<float>(a, stream);
    case MB200_BF16: return fwd_of<__nv_bfloat16>(a, stream);
    default: return fwd_of<__half>(a, stream);
  }
}

cudaError_t launch_gated_scan_bwd(const GatedScanArgs& a, int dtype, float* dA, cudaStream_t stream) {
  if (a.dim == 0) return cudaSuccess;
  if (a.batch > 0) {
    cudaError_t e;
    switch (dtype) {
      case MB200_F32: e = bwd_of<float>(a, stream); break;
      case MB200_BF16: e = bwd_of<__nv_bfloat16>(a, stream); break;
      default: e = bwd_of<__half>(a, stream); break;
    }
    if (e != cudaSuccess) return e;
    note_launches(1);
    if (a.batch == 1) return cudaSuccess;  // part is dA
  }
  note_launches(1);
  gated_reduce_kernel<<<(unsigned)((a.dim + 127) / 128), 128, 0, stream>>>(a.part, a.batch, a.dim, dA);
  return cudaGetLastError();
}

cudaError_t launch_gated_step(const GatedStepArgs& a, int dtype, int state_dtype, cudaStream_t stream) {
  if (a.batch * a.dim == 0) return cudaSuccess;
  note_launches(1);
  const bool wide = state_dtype == MB200_F32;
  switch (dtype) {
    case MB200_F32: return step_of<float, float>(a, stream);
    case MB200_BF16:
      return wide ? step_of<__nv_bfloat16, float>(a, stream) : step_of<__nv_bfloat16, __nv_bfloat16>(a, stream);
    default: return wide ? step_of<__half, float>(a, stream) : step_of<__half, __half>(a, stream);
  }
}

}  // namespace mb200
