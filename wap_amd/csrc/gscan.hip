// Gated linear recurrence over a sequence, forward, backward and one step.
//
//   z_t = sigmoid(gz_t), n_t = tanh(gn_t)          gates packed [z|n]
//   h_t = (1 - z_t) n_t + z_t h_{t-1}              masked step: h_t = h_{t-1}
//
// The blend is the GRU's; its gates do not see the state, so h is linear in
// the state before: a run of steps is h_out = A h_in + B, and runs compose.
// The state, the gates and all sums are f32; h is rounded once, where it is
// stored.
//
// Layout.  A workgroup takes a tile of S = W R steps by 64 VEC channels: each
// of its W waves holds R steps in registers (one load of every gate, all of
// them in flight together), reduces them to (A, B) and finds the state before
// them from the waves before it (LDS) and the tiles before its own.  Tiles of
// one channel block are chained through global memory in one launch, so that
// gates are read once and h is written once: what a chunked scan of two
// launches reads twice.
//
// The chain.  A tile publishes (A, B) of its steps, looks at as many tiles
// before it as it has waves until the end state of one of them is there and
// the runs of all between, steps over those, and publishes its own end state.
// The end state is fma(A, state before, B) whichever tile the walk began at, so
// results do not depend on timing.  Every published word shows by itself
// whether it has been written (a pattern of ones, a NaN that no result has,
// stands for "not yet"), so no flag has to be ordered against data; words are
// read and written with device-scope atomics, since the eight XCDs' L2 caches
// are not coherent.  A tile waits only for tiles of earlier tickets, and a
// ticket is drawn by a workgroup that is running already: every wait ends.
#include <hip/hip_runtime.h>

#include "opcommon.h"

namespace {

using namespace wap;

struct Gates {
  float z, zc, n;  // z, 1 - z (from the exponential: no cancellation), n
};

// exp(SCALE x), SCALE a power of two; with CUT at most 2^126, which keeps what
// it is multiplied with finite.  For 16-bit gates one multiplication and the
// hardware's exp2 (relative error |x| 2^-24) are far below the gates' own
// rounding; f32 gates add what the product lost.
template <typename T, int SCALE, bool CUT>
__device__ __forceinline__ float exp_of(float x) {
  constexpr float log2e = SCALE * 1.44269502162933349609375f;
  float t = x * log2e;
  // the smaller one, NaN if x is NaN
  if constexpr (CUT) t = __builtin_elementwise_minimum(t, 126.f);
  const float e = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(T) == 4) {
    // SCALE x log2 e - t, with log2 e in two parts; not where t is cut or e ends
    const float lost = fmaf(x, SCALE * 1.92596299112661746887e-8f,
                            fmaf(x, log2e, -t));
    return fabsf(t) < 120.f ? fmaf(e * 0.693147180559945309f, lost, e) : e;
  }
  return e;
}

// z = 1 / (1 + e), 1 - z = e z with e = exp(-gz), cut at 2^126 so that the
// product stays finite; where it is cut z is 0.  tanh x = 1 - 2 / (1 + exp(2
// x)), absolute error 1.2e-7; near zero, where that is not enough, the odd
// series: to x^5 below 0.1 (the next term is 6e-8 of the value there), for f32
// gates to x^9 below 0.3 (5e-8).
template <typename T>
__device__ __forceinline__ Gates gates(float gz, float gn) {
  const float e = exp_of<T, -1, true>(gz);
  Gates r;
  const float z = __builtin_amdgcn_rcpf(1.f + e);
  r.zc = e * z;
  r.z = e >= 0x1p126f ? 0.f : z;  // NaN stays
  const float f = exp_of<T, 2, false>(gn);
  const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + f), 1.f);
  const float q = gn * gn;
  constexpr bool wide = sizeof(T) == 4;
  float p = fmaf(q, 2.f / 15.f, -1.f / 3.f);
  if constexpr (wide)
    p = fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f),
             -1.f / 3.f);
  const float near = gn * fmaf(q, p, 1.f);
  r.n = __builtin_unpredictable(fabsf(gn) < (wide ? 0.3f : 0.1f)) ? near : far;
  return r;
}

// ------------------------------------------------------------ the chain

constexpr uint32_t UNSET = 0xffffffffu;

struct Chain {
  uint64_t* run;     // (A, B) of every tile's steps
  uint32_t* end;     // end state of every tile
  uint32_t* ticket;  // one counter a group, 128 bytes apart; null: one tile
  int blocks;        // channel blocks of all sequences
  int groups, per;   // blocks are dealt to groups, `per` to each at most
  int tiles;         // tiles of one sequence
};

// A result's bits: any NaN becomes one that is not the pattern for "not yet".
__device__ __forceinline__ uint32_t word(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0x7fc00000u : u;
}

template <typename W>
__device__ __forceinline__ W peek(const W* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename W>
__device__ __forceinline__ void post(W* p, W v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The next tile of this workgroup's group, in time order over all channel
// blocks of the group: (block, place in time). False: none.
// The grid has groups * per * tiles workgroups and blockIdx % groups is the
// group, so that with workgroups dealt to the eight XCDs in turn a chain stays
// on one XCD.  Groups of one XCD take blocks side by side: where rows are no
// multiple of a cache line, the lines that two blocks share then come from one
// L2.
__device__ __forceinline__ bool next_tile(const Chain& ch, int* block,
                                          int* at) {
  const int grp = blockIdx.x % ch.groups;
  int k = blockIdx.x / ch.groups;  // same in every lane: kept in scalars
  if (ch.ticket) {
    __shared__ int drawn;
    if (threadIdx.x == 0)
      drawn = (int)__hip_atomic_fetch_add(ch.ticket + grp * 32, 1u,
                                          __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    k = __builtin_amdgcn_readfirstlane(drawn);
  }
  *at = k / ch.per;
  // (4 x 8000 x 1001 f32 forward 99.5 us, 108 in the groups' own order)
  const int side =
      ch.groups % 8 ? grp : grp % 8 * (ch.groups / 8) + grp / 8;
  *block = k % ch.per * ch.groups + side;
  return *block < ch.blocks;
}

// Tiles of fewer waves hold their whole sequence.
template <int W>
constexpr bool may_chain = W >= 8;

// What the waves of a workgroup have seen of the tiles before theirs.
template <int VEC, int W>
struct Seen {
  float end[W][64 * VEC];
  float2 run[W][64 * VEC];
  int has[2][W];  // 1: the end state, 2: the run; by turns
};

// A wave's place in the words of tile `at`; tiles are `stride` apart.
template <int VEC>
__device__ __forceinline__ long words_at(const Chain& ch, int block, int at,
                                         int lane) {
  return ((long)at * ch.blocks + block) * (64 * VEC) + lane * VEC;
}

// One wave publishes the run (A, B) of its tile's steps.  Nobody steps over
// the first tile, which publishes its end state at once, or over the last.
template <int VEC>
__device__ __forceinline__ void publish(const Chain& ch, int block, int at,
                                        int lane, const float (&A)[VEC],
                                        const float (&B)[VEC]) {
  if (at == 0 || at + 1 == ch.tiles) return;
  uint64_t* p = ch.run + words_at<VEC>(ch, block, at, lane);
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    post(p + j, (uint64_t)word(A[j]) | (uint64_t)word(B[j]) << 32);
}

// The whole workgroup finds the state h before tile `at` (tile 0: h as it is)
// and publishes the state after it; A and B count in wave 0.  Wave w looks at
// tile at-1-w, so that a workgroup steps over W tiles in one round trip to
// memory and holds few registers for it.
template <int VEC, int W>
__device__ __forceinline__ void walk(const Chain& ch, int block, int at,
                                     int wave, int lane, const float (&A)[VEC],
                                     const float (&B)[VEC],
                                     Seen<VEC, W>& seen, float (&h)[VEC]) {
  const long stride = (long)ch.blocks * (64 * VEC);  // from tile to tile
  const long mine = words_at<VEC>(ch, block, at, lane);
  if (at > 0) {
    const int reach = at < W ? at : W;
    const long p = mine - (wave + 1) * stride;  // read where wave < reach
    int has = 0;
    int from = -1;  // the nearest tile before this one whose end is there
    for (int turn = 0;; turn ^= 1) {
      if (wave < reach && !(has & 1)) {
        // the end first: where it is there the run is not needed, and where it
        // is not there is time
        uint32_t e[VEC];
        bool there = true;
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = peek(ch.end + p + j);
#pragma unroll
        for (int j = 0; j < VEC; ++j) there &= e[j] != UNSET;
        if (__all(there)) {
          has |= 1;
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            seen.end[wave][lane * VEC + j] = __uint_as_float(e[j]);
        } else if (wave + 1 < reach && !(has & 2)) {
          // (the end of the last tile in reach is not stepped over)
          uint64_t r[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) r[j] = peek(ch.run + p + j);
          there = true;
#pragma unroll
          for (int j = 0; j < VEC; ++j) there &= (uint32_t)r[j] != UNSET;
          if (__all(there)) {
            has |= 2;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              seen.run[wave][lane * VEC + j] =
                  make_float2(__uint_as_float((uint32_t)r[j]),
                              __uint_as_float((uint32_t)(r[j] >> 32)));
          }
        }
      }
      if (lane == 0) seen.has[turn][wave] = has;
      __syncthreads();
      // every wave comes to the same answer; the next turn writes elsewhere
#pragma unroll
      for (int i = W - 1; i >= 0; --i) {
        const int q = seen.has[turn][i];
        if (i < reach) from = q & 1 ? i : q & 2 ? from : -1;
      }
      from = __builtin_amdgcn_readfirstlane(from);
      if (from >= 0) break;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] = seen.end[from][lane * VEC + j];
    for (int i = from - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 q = seen.run[i][lane * VEC + j];
        h[j] = fmaf(q.x, h[j], q.y);
      }
  }
  if (wave == 0 && at + 1 < ch.tiles) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      post(ch.end + mine + j, word(fmaf(A[j], h[j], B[j])));
  }
}

// "Not yet" everywhere, and the tickets at zero.
__global__ void chain_clear_kernel(uint4* __restrict__ words, long n,
                                   uint32_t* __restrict__ ticket, int m) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) words[i] = make_uint4(UNSET, UNSET, UNSET, UNSET);
  if (i < m) ticket[i] = 0u;
}

// ------------------------------------------------------------ forward

struct Scan {
  long gsb, gst;      // strides of g over sequence and time
  long dsb, dst;      // strides of dh
  const float* h0;    // [B, D] or null
  const float* mask;  // [B, L] or null
  long L;
  int D, dblocks;     // channel blocks of one sequence
};

// The forward pass leaves the state before step MARK, 2 MARK, .. for the
// backward pass, whose tiles begin at such steps: f32, 1 / MARK of the size of
// h, and each pass can cut time as suits it.
constexpr int MARK = 64;

__host__ __device__ __forceinline__ long marks_of(long L) {
  return (L - 1) / MARK;
}

// Which of this wave's steps exist and count, one bit each.
template <int ROWS>
__device__ __forceinline__ constexpr uint32_t all_steps() {
  return (1u << ROWS) - 1;
}

template <int ROWS>
__device__ __forceinline__ uint32_t steps_on(const Scan& s, long b, long t0,
                                             int lane) {
  bool on = lane < ROWS && t0 + lane < s.L;
  if (on && s.mask) on = s.mask[b * s.L + t0 + lane] > 0.f;
  return (uint32_t)__ballot(on);
}

// A lane's place in a row that is the same in all lanes: the row's address
// stays in scalar registers, opaque to the compiler, which would otherwise add
// it up in 64-bit vector work for every access, and the lane's 32-bit byte
// offset is part of the instruction.
template <typename T>
using Global = __attribute__((address_space(1))) T*;

template <typename V, typename T>
__device__ __forceinline__ Global<V> lane_at(T* row, uint32_t bytes) {
  typedef std::conditional_t<std::is_const_v<T>, const char, char> byte;
  Global<byte> p = (Global<byte>)row;
  asm("" : "+s"(p));
  return (Global<V>)(p + bytes);
}

// COLD: past the caches, where a pass moves more than the 256 MB of the last
// one, so that none of it would be there for the next reader (8 x 8192 x 2048
// bf16: forward 172 us, 178 without, backward 302, 312).  Not where channel
// blocks share cache lines: the caches put those together (4 x 8000 x 1001
// f32: forward 92 us, with cold stores 99, with cold loads too 108).
template <bool COLD, typename V, typename T>
__device__ __forceinline__ void put(T* row, uint32_t bytes, const V& v) {
  if constexpr (COLD)
    __builtin_nontemporal_store(v, lane_at<V>(row, bytes));
  else
    *lane_at<V>(row, bytes) = v;
}

// Rows of a wave, kept as they came (two 16-bit values a register).  Rows past
// the end read the last one; what is read there is not used.
template <typename T, int VEC>
using Pack = typename VecOf<T, VEC, sizeof(T)>::type;

// ROWS + 1 stands for more than ROWS.
template <int ROWS>
__device__ __forceinline__ int rows_left(long n) {
  return n > ROWS ? ROWS + 1 : n < 0 ? 0 : (int)n;
}

template <bool COLD, typename T, int VEC, int ROWS>
__device__ __forceinline__ void load_rows(const T* base, uint32_t bytes,
                                          long stride, int rows,
                                          Pack<T, VEC> (&v)[ROWS]) {
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if constexpr (COLD)
      v[r] = __builtin_nontemporal_load(
          lane_at<const Pack<T, VEC>>(base, bytes));
    else
      v[r] = *lane_at<const Pack<T, VEC>>(base, bytes);
    if (r + 1 < rows) base += stride;
  }
}

template <typename T, int VEC, int W, int ROWS, bool COLD>
__global__ __launch_bounds__(64 * W) void gscan_fwd_kernel(
    const T* __restrict__ g, Scan s, Chain ch, T* __restrict__ out,
    float* __restrict__ last, float* __restrict__ marks) {
  constexpr int CH = 64 * VEC;
  __shared__ float2 runs[W][CH];
  __shared__ Seen<VEC, may_chain<W> ? W : 1> seen;
  const bool chained = may_chain<W> && ch.tiles > 1;
  int block, at;
  if (!next_tile(ch, &block, &at)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long b = block / s.dblocks;
  const int d = block % s.dblocks * CH + lane * VEC;
  // lanes past the last channel read its place and store nothing
  const bool inside = d < s.D;
  const uint32_t dc = inside ? d : s.D - VEC;
  const uint32_t off = dc * (uint32_t)sizeof(T);
  const long t0 = ((long)at * W + wave) * ROWS;
  const uint32_t on = steps_on<ROWS>(s, b, t0, lane);
  const int rows = rows_left<ROWS>(s.L - t0);
  float h[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    h[j] = s.h0 && at == 0 ? s.h0[b * s.D + dc + j] : 0.f;
  float a[ROWS][VEC], x[ROWS][VEC];
  // a wave whose steps are all masked reads none of them; short sequences do
  // not wait for the mask to know
  if (chained ? on != 0 : rows > 0) {
    Pack<T, VEC> rz[ROWS], rn[ROWS];
    const T* p = g + b * s.gsb + t0 * s.gst;
    load_rows<COLD, T, VEC, ROWS>(p, off, s.gst, rows, rz);
    load_rows<COLD, T, VEC, ROWS>(p + s.D, off, s.gst, rows, rn);
    // all loads leave before the first value is used
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const Gates q = gates<T>((float)rz[r][j], (float)rn[r][j]);
        a[r][j] = q.z;
        x[r][j] = q.zc * q.n;
      }
  }
  if (on != all_steps<ROWS>()) {  // same in every lane
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (!(on >> r & 1)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[r][j] = 1.f, x[r][j] = 0.f;
      }
  }
  // step r becomes the run of the wave's steps up to r
#pragma unroll
  for (int r = 1; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[r][j] = fmaf(a[r][j], x[r - 1][j], x[r][j]);
      a[r][j] *= a[r - 1][j];
    }
  if constexpr (W > 1) {
    float A[VEC], B[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      A[j] = a[ROWS - 1][j], B[j] = x[ROWS - 1][j];
      runs[wave][lane * VEC + j] = make_float2(A[j], B[j]);
    }
    __syncthreads();
    if (chained) {
      if (wave == 0) {
        for (int w = 1; w < W; ++w)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float2 q = runs[w][lane * VEC + j];
            A[j] *= q.x;
            B[j] = fmaf(q.x, B[j], q.y);
          }
        publish<VEC>(ch, block, at, lane, A, B);
      }
      if constexpr (may_chain<W>)
        walk<VEC, W>(ch, block, at, wave, lane, A, B, seen, h);
    }
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 q = runs[w][lane * VEC + j];
        h[j] = fmaf(q.x, h[j], q.y);
      }
  }
  if (marks && t0 % MARK == 0 && t0 > 0 && inside && rows > 0) {
    float* m = marks + (b * marks_of(s.L) + t0 / MARK - 1) * s.D + d;
#pragma unroll
    for (int j = 0; j < VEC; ++j) m[j] = h[j];
  }
  T* o = out + (b * s.L + t0) * s.D;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    Pack<T, VEC> v;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (T)fmaf(a[r][j], h[j], x[r][j]);
    if (r < rows && inside) put<COLD>(o, off, v);
    o += s.D;
  }
  // steps past the end leave the state as it is
  if (inside && rows > 0 && rows <= ROWS) {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      last[b * s.D + d + j] = fmaf(a[ROWS - 1][j], h[j], x[ROWS - 1][j]);
  }
}

// ------------------------------------------------------------ backward
//
//   delta_t = dh_t + z_{t+1} delta_{t+1}           (dlast joins the last one)
//   dgz = delta (h_{t-1} - n) z (1 - z),  dgn = delta (1 - z) (1 - n^2)
//
// With c_t = z_t delta_t, the gradient that leaves step t for the state before
// it, c_t = z_t (c_{t+1} + dh_t): the same chain, from the end.  The states
// are made again from the states that the forward pass left, which reads less
// than h itself would be, and has them in f32.

template <typename T, int VEC, int W, int ROWS, bool COLD>
__global__ __launch_bounds__(64 * W) void gscan_bwd_kernel(
    const T* __restrict__ g, Scan s, Chain ch, const float* __restrict__ marks,
    const T* __restrict__ dh, const float* __restrict__ dlast,
    T* __restrict__ dg, float* __restrict__ dh0) {
  constexpr int CH = 64 * VEC;
  __shared__ float2 runs[W][CH];
  __shared__ float back[W][CH];
  __shared__ Seen<VEC, may_chain<W> ? W : 1> seen;
  const bool chained = may_chain<W> && ch.tiles > 1;
  int block, from_end;
  if (!next_tile(ch, &block, &from_end)) return;
  const int at = ch.tiles - 1 - from_end;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long b = block / s.dblocks;
  const int d = block % s.dblocks * CH + lane * VEC;
  const bool inside = d < s.D;
  const uint32_t dc = inside ? d : s.D - VEC;
  const uint32_t off = dc * (uint32_t)sizeof(T);
  const long t0 = ((long)at * W + wave) * ROWS;
  const int rows = rows_left<ROWS>(s.L - t0);
  const uint32_t on = steps_on<ROWS>(s, b, t0, lane);
  float z[ROWS][VEC], zc[ROWS][VEC], n[ROWS][VEC];
  Pack<T, VEC> ru[ROWS];  // dh stays as it came: half the registers for 16 bits
  if (dh && rows > 0)
    load_rows<COLD, T, VEC, ROWS>(dh + b * s.dsb + t0 * s.dst, off, s.dst, rows,
                                  ru);
  if (on) {
    Pack<T, VEC> rz[ROWS], rn[ROWS];
    const T* p = g + b * s.gsb + t0 * s.gst;
    load_rows<COLD, T, VEC, ROWS>(p, off, s.gst, rows, rz);
    load_rows<COLD, T, VEC, ROWS>(p + s.D, off, s.gst, rows, rn);
    // all loads leave before the first value is used
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const Gates q = gates<T>((float)rz[r][j], (float)rn[r][j]);
        z[r][j] = q.z;
        zc[r][j] = q.zc;
        n[r][j] = q.n;
      }
  }
  if (on != all_steps<ROWS>()) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (!(on >> r & 1)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[r][j] = 1.f, zc[r][j] = n[r][j] = 0.f;
      }
  }
  if (!dh || rows < ROWS) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (!dh || r >= rows) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) ru[r][j] = (T)0.f;
      }
  }
  float h[VEC], c[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    // (every wave takes its tile's first state and steps to its own)
    h[j] = at > 0 ? marks[(b * marks_of(s.L) + (long)at * W * ROWS / MARK - 1) *
                              s.D + dc + j]
           : s.h0 ? s.h0[b * s.D + dc + j]
                  : 0.f;
    c[j] = dlast ? dlast[b * s.D + dc + j] : 0.f;
  }
  float A[VEC], C[VEC];
  if constexpr (W > 1) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float B = 0.f;
      A[j] = 1.f, C[j] = 0.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        A[j] *= z[r][j];
        B = fmaf(z[r][j], B, zc[r][j] * n[r][j]);
      }
#pragma unroll
      for (int r = ROWS - 1; r >= 0; --r)
        C[j] = z[r][j] * (C[j] + (float)ru[r][j]);
      runs[wave][lane * VEC + j] = make_float2(A[j], B);
      back[wave][lane * VEC + j] = C[j];
    }
    __syncthreads();
    if (chained) {
      if (wave == 0) {
        // the waves' runs from the end; this one's own is the last
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float a = 1.f, b = 0.f;
          for (int w = W - 1; w > 0; --w) {
            const float q = runs[w][lane * VEC + j].x;
            a *= q;
            b = fmaf(q, b, back[w][lane * VEC + j]);
          }
          C[j] = fmaf(A[j], b, C[j]);
          A[j] *= a;
        }
        publish<VEC>(ch, block, from_end, lane, A, C);
      }
    }
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 q = runs[w][lane * VEC + j];
        h[j] = fmaf(q.x, h[j], q.y);
      }
  }
  // what delta is multiplied by needs the states alone: made while the chain
  // from the end is on its way, in the place of 1 - z and n
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float past = h[j], q = zc[r][j], m = n[r][j];
      h[j] = fmaf(z[r][j], past, q * m);
      zc[r][j] = q * z[r][j] * (past - m);
      n[r][j] = q * fmaf(-m, m, 1.f);
    }
  if constexpr (W > 1) {
    if constexpr (may_chain<W>)
      if (chained)
        walk<VEC, W>(ch, block, from_end, wave, lane, A, C, seen, c);
    for (int w = W - 1; w > wave; --w)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        c[j] = fmaf(runs[w][lane * VEC + j].x, c[j], back[w][lane * VEC + j]);
  }
  T* o = dg + (b * s.L + t0 + ROWS) * 2 * s.D;
#pragma unroll
  for (int r = ROWS - 1; r >= 0; --r) {
    float fz[VEC], fn[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float delta = c[j] + (float)ru[r][j];
      fz[j] = delta * zc[r][j];
      fn[j] = delta * n[r][j];
      c[j] = z[r][j] * delta;
    }
    // a step that does not count has no gradient, whatever passes it by
    if (!(on >> r & 1)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) fz[j] = fn[j] = 0.f;
    }
    o -= 2 * (long)s.D;
    if (r < rows && inside) {
      Pack<T, VEC> vz, vn;
#pragma unroll
      for (int j = 0; j < VEC; ++j) vz[j] = (T)fz[j], vn[j] = (T)fn[j];
      put<COLD>(o, off, vz);
      put<COLD>(o + s.D, off, vn);
    }
  }
  if (dh0 && inside && t0 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) dh0[b * s.D + d + j] = c[j];
  }
}

// ------------------------------------------------------------ one token

template <typename T>
__global__ void gstep_kernel(
    const T* __restrict__ g, long gsb, const float* __restrict__ h,
    T* __restrict__ out, float* __restrict__ h_new, long total, int D) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const long b = i / D, d = i % D;
  const T* p = g + b * gsb + d;
  const Gates q = gates<T>((float)p[0], (float)p[D]);
  const float v = fmaf(q.z, h[i], q.zc * q.n);
  h_new[i] = v;
  out[i] = (T)v;
}

// ------------------------------------------------------------ host

void check_gates(const torch::Tensor& g, int dim) {
  TORCH_CHECK(g.is_cuda(), "gated_scan: g must be on the GPU");
  TORCH_CHECK(g.dim() == dim && g.size(-1) % 2 == 0 && g.stride(-1) == 1,
              "gated_scan: g must end in a dense axis of 2 D");
  TORCH_CHECK(g.size(-1) / 2 < (1 << 29) && g.numel() > 0,
              "gated_scan: empty or too wide");
}

void check_state(const c10::optional<torch::Tensor>& h,
                 const torch::Tensor& g) {
  if (!h.has_value()) return;
  WAP_F32(*h, g, "gated_scan");
  TORCH_CHECK(h->dim() == 2 && h->size(0) == g.size(0) &&
                  h->size(1) == g.size(-1) / 2,
              "gated_scan: a state must be [B, D]");
}

void check_mask(const c10::optional<torch::Tensor>& mask,
                const torch::Tensor& g) {
  if (!mask.has_value()) return;
  WAP_F32(*mask, g, "gated_scan");
  TORCH_CHECK(mask->dim() == 2 && mask->size(0) == g.size(0) &&
                  mask->size(1) == g.size(1),
              "gated_scan: mask must be [B, T]");
}

// Channels of a lane, waves of a workgroup, steps of a wave.
struct Shape {
  int vec, waves, rows;
};

// How a pass is cut, by the number of 64-channel blocks and the length (us on
// an MI355X, a call among others; "2,8,16": two channels a lane, 8 waves of 16
// steps).
// - Up to 256 steps one tile holds the sequence, and nothing is chained: 16 x
//   200 x 256 bf16 forward 7.9 in one tile of 1,16,16, 10.4 in two of 1,8,16.
// - Few blocks: time is the only axis to spread over, and a round trip of the
//   chain should step far: 1 x 40000 x 128 bf16 forward 27 with tiles of 256
//   steps, 55 with 128; from 5 blocks on 128 (2 x 20000 x 512: 51, 45).
// - Two channels a lane where that leaves enough workgroups, from 64 blocks on
//   (short sequences, all latency, from 128): 32 x 4096 x 256 bf16 forward 53,
//   with one 65; 4 x 8192 x 1500: 79, 119; with 32 blocks, 8 x 4096 x 256, 20,
//   21; 16 x 200 x 256: 10.2, 7.9.  The backward pass then holds 8 steps a wave,
//   to stay under 128 registers: 8 x 8192 x 2048 302, with 16 steps of one
//   channel 320.
Shape shape_of(const torch::Tensor& g, bool backward) {
  const long L = g.size(1), D = g.size(2) / 2;
  const long blocks = g.size(0) * ((D + 63) / 64);
  const bool two = blocks >= (L > 256 ? 64 : 128) && D % 2 == 0 &&
                   g.element_size() == 2;
  const int rows = L <= 8 || (backward && two) ? 8 : 16;
  if (backward && two && L > 64 && L <= 256)  // no room for 16 steps of two
    return {1, L <= 128 ? 8 : 16, 16};
  if (L <= (backward && two ? 64 : 16 * rows)) {
    int w = 1;
    while (w * rows < L) w *= 2;
    return {two ? 2 : 1, w, rows};
  }
  return {two ? 2 : 1, blocks < 5 ? 16 : 8, rows};
}

struct Cut {
  Shape p;
  Chain ch;
  long words;  // published words of one kind
  Scan s;
};

Cut cut_of(const torch::Tensor& g, const c10::optional<torch::Tensor>& h0,
           const c10::optional<torch::Tensor>& mask, bool backward) {
  Cut c;
  c.s.gsb = g.stride(0);
  c.s.gst = g.stride(1);
  c.s.dsb = c.s.dst = 0;
  c.s.h0 = data_or_null<float>(h0);
  c.s.mask = data_or_null<float>(mask);
  c.s.L = g.size(1);
  c.s.D = g.size(2) / 2;
  c.p = shape_of(g, backward);
  const int wide = 64 * c.p.vec;
  c.s.dblocks = (c.s.D + wide - 1) / wide;
  const long blocks = (long)g.size(0) * c.s.dblocks;
  const long step = (long)c.p.waves * c.p.rows;
  const long tiles = (c.s.L + step - 1) / step;
  TORCH_CHECK(blocks < (1L << 30) && tiles < (1L << 30),
              "gated_scan: too many sequences, channels or steps");
  TORCH_CHECK(tiles == 1 || c.p.waves >= 8, "gated_scan: no such shape");
  c.ch.blocks = blocks;
  c.ch.tiles = tiles;
  c.ch.groups = tiles == 1 ? 1 : std::min(blocks, 64L);
  c.ch.per = (blocks + c.ch.groups - 1) / c.ch.groups;
  TORCH_CHECK((long)c.ch.groups * c.ch.per * tiles < (1L << 31),
              "gated_scan: too many tiles");
  c.ch.run = nullptr;
  c.ch.end = nullptr;
  c.ch.ticket = nullptr;
  c.words = blocks * tiles * wide;
  return c;
}

// Words of the chain, cleared: end states | runs | tickets.
torch::Tensor make_chain(const torch::Tensor& g, Cut* c) {
  const auto opts = g.options().dtype(at::kInt);
  const long tickets = c->ch.groups * 32L;
  auto buf = torch::empty({3 * c->words + tickets}, opts);
  uint32_t* p = data<uint32_t>(buf);
  c->ch.end = p;
  c->ch.run = reinterpret_cast<uint64_t*>(p + c->words);
  c->ch.ticket = p + 3 * c->words;
  const long quads = 3 * c->words / 4;  // words is a multiple of 64
  const long n = std::max(quads, tickets);
  hipLaunchKernelGGL(chain_clear_kernel, dim3((n + 255) / 256), dim3(256), 0,
                     stream_of(g), reinterpret_cast<uint4*>(p), quads,
                     c->ch.ticket, (int)tickets);
  launched("gated_scan");
  return buf;
}

// Whether channel blocks share no cache line.
bool in_lines(const torch::Tensor& t, long D) {
  const long line = 128 / t.element_size();
  return D % line == 0 && t.stride(0) % line == 0 && t.stride(1) % line == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 128 == 0;
}

template <int VEC, int W, int ROWS>
struct Fixed {
  static constexpr int vec = VEC, waves = W, rows = ROWS;
};

// f(Fixed<...>) for a shape that shape_of gives.
template <typename T, bool BACKWARD, typename F>
void by_shape(const Shape& p, F&& f) {
  if constexpr (sizeof(T) == 2) {
    if (p.vec == 2) {
      constexpr int R = BACKWARD ? 8 : 16;
      if (p.waves == 1 && p.rows == 8) return f(Fixed<2, 1, 8>());
      switch (p.waves) {
        case 1: return f(Fixed<2, 1, R>());
        case 2: return f(Fixed<2, 2, R>());
        case 4: return f(Fixed<2, 4, R>());
        case 8: return f(Fixed<2, 8, R>());
      }
      if constexpr (!BACKWARD) return f(Fixed<2, 16, R>());
      TORCH_CHECK(false, "gated_scan: no such shape");
    }
  }
  if (p.rows == 8) return f(Fixed<1, 1, 8>());
  switch (p.waves) {
    case 1: return f(Fixed<1, 1, 16>());
    case 2: return f(Fixed<1, 2, 16>());
    case 4: return f(Fixed<1, 4, 16>());
    case 8: return f(Fixed<1, 8, 16>());
    default: return f(Fixed<1, 16, 16>());
  }
}

}  // namespace

// -> h, last state and, with `keep` and where the backward pass takes more
// than one tile, the states that it begins from.
std::vector<torch::Tensor> gated_scan_fwd(
    torch::Tensor g, c10::optional<torch::Tensor> h0,
    c10::optional<torch::Tensor> mask, bool keep) {
  check_gates(g, 3);
  check_state(h0, g);
  check_mask(mask, g);
  c10::DeviceGuard guard(g.device());
  const long B = g.size(0), L = g.size(1), D = g.size(2) / 2;
  auto out = torch::empty({B, L, D}, g.options());
  auto last = torch::empty({B, D}, g.options().dtype(at::kFloat));
  Cut c = cut_of(g, h0, mask, false);
  torch::Tensor buf, marks;
  if (c.ch.tiles > 1) buf = make_chain(g, &c);
  const Shape back = shape_of(g, true);
  if (keep && L > (long)back.waves * back.rows)
    marks = torch::empty({B, marks_of(L), D}, last.options());
  const dim3 grid((long)c.ch.groups * c.ch.per * c.ch.tiles);
  const bool cold =
      3 * out.numel() * out.element_size() > (256L << 20) && in_lines(g, D);
  by_type(g, "gated_scan", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_shape<T, false>(c.p, [&](auto p) {
      constexpr int V = decltype(p)::vec, W = decltype(p)::waves,
                    R = decltype(p)::rows;
      auto go = [&](auto past) {
        hipLaunchKernelGGL(
            (gscan_fwd_kernel<T, V, W, R, decltype(past)::value>), grid,
            dim3(64 * W), 0, stream_of(g), data<T>(g), c.s, c.ch, data<T>(out), data<float>(last),
            marks.defined() ? data<float>(marks) : nullptr);
      };
      if (cold)
        go(std::true_type());
      else
        go(std::false_type());
    });
  });
  launched("gated_scan");
  if (marks.defined()) return {out, last, marks};
  return {out, last};
}

std::vector<torch::Tensor> gated_scan_bwd(
    torch::Tensor g, c10::optional<torch::Tensor> h0,
    c10::optional<torch::Tensor> mask, c10::optional<torch::Tensor> marks,
    c10::optional<torch::Tensor> dh, c10::optional<torch::Tensor> dlast) {
  check_gates(g, 3);
  check_state(h0, g);
  check_state(dlast, g);
  check_mask(mask, g);
  const long B = g.size(0), L = g.size(1), D = g.size(2) / 2;
  if (dh.has_value())
    TORCH_CHECK(dh->scalar_type() == g.scalar_type() &&
                    dh->device() == g.device() && dh->dim() == 3 &&
                    dh->size(0) == B && dh->size(1) == L &&
                    dh->size(2) == D && (dh->stride(2) == 1 || D == 1),
                "gated_scan: dh must be [B, T, D] in g's type");
  c10::DeviceGuard guard(g.device());
  auto dg = torch::empty({B, L, 2 * D}, g.options());
  torch::Tensor dh0;
  if (h0.has_value()) dh0 = torch::empty_like(*h0);
  Cut c = cut_of(g, h0, mask, true);
  if (dh.has_value()) {
    c.s.dsb = dh->stride(0);
    c.s.dst = dh->stride(1);
  }
  torch::Tensor buf;
  if (c.ch.tiles > 1) {
    TORCH_CHECK(marks.has_value(), "gated_scan: the forward pass's states are "
                                   "missing");
    WAP_F32(*marks, g, "gated_scan");
    TORCH_CHECK(marks->numel() == B * marks_of(L) * D &&
                    c.p.waves * c.p.rows % MARK == 0,
                "gated_scan: the forward pass's states are of another shape");
    buf = make_chain(g, &c);
  }
  const dim3 grid((long)c.ch.groups * c.ch.per * c.ch.tiles);
  const bool cold =
      5 * (dg.numel() / 2) * dg.element_size() > (256L << 20) &&
      in_lines(g, D) && (!dh.has_value() || in_lines(*dh, D));
  by_type(g, "gated_scan", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    by_shape<T, true>(c.p, [&](auto p) {
      constexpr int V = decltype(p)::vec, W = decltype(p)::waves,
                    R = decltype(p)::rows;
      auto go = [&](auto past) {
        hipLaunchKernelGGL(
            (gscan_bwd_kernel<T, V, W, R, decltype(past)::value>), grid,
            dim3(64 * W), 0, stream_of(g), data<T>(g), c.s, c.ch,
            data_or_null<float>(marks), data_or_null<T>(dh), data_or_null<float>(dlast), data<T>(dg),
            dh0.defined() ? data<float>(dh0) : nullptr);
      };
      if (cold)
        go(std::true_type());
      else
        go(std::false_type());
    });
  });
  launched("gated_scan backward");
  if (dh0.defined()) return {dg, dh0};
  return {dg};
}

std::tuple<torch::Tensor, torch::Tensor> gated_step_run(torch::Tensor g,
                                                        torch::Tensor h) {
  check_gates(g, 2);
  check_state(h, g);
  c10::DeviceGuard guard(g.device());
  const long total = h.numel();
  const int D = h.size(1);
  auto out = torch::empty_like(h, g.options());
  auto h_new = torch::empty_like(h);
  by_type(g, "gated_step", [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(gstep_kernel<T>, dim3((total + 255) / 256), dim3(256),
                       0, stream_of(g), data<T>(g), g.stride(0),
                       data<float>(h), data<T>(out), data<float>(h_new), total,
                       D);
  });
  launched("gated_step");
  return {out, h_new};
}
