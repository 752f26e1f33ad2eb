// Attention over packed sequences for gfx950: forward and backward.
//
// q [T, H, D], k and v [T, HK, D] hold the sequences one behind the other;
// sequence i is rows cu[i]..cu[i+1], of which the first lengths[i] are
// tokens and the rest padding.  Per head, with the keys j that row i sees:
//   s = scale q.k,  p = exp(s - lse),  lse = log sum exp(s),  o = p v
//   dV = p^T dO,  dP = dO v^T,  dS = p (dP - D),  D = dO.o
//   dQ = scale dS k,  dK = scale dS^T q  (backward computes p again from lse)
//
// Matrix work is v_mfma_f32_32x32x16.  Its accumulator holds, in lane l,
// column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4: a product whose
// operands are swapped so that the softmax's row is the COLUMN leaves every
// lane with 16 values of one row.  Its maximum and sum need one exchange
// between lanes l and l ^ 32, and the 16 values, rounded, ARE the second
// product's B operand if that product takes its reduction in the order in
// which they stand.  Its A operand comes out of LDS through transposing
// reads of 4 neighbouring rows, which give exactly that order.  So
// probabilities never pass through LDS, and no transposed copy is made.
//
// Sequences are found on the GPU: a call waits for nothing and can be
// captured.  A tile of R rows lies in one sequence; sequence i of those that
// begin at b[i] owns the slots from b[i] / R + i on, which is at least as many
// as it has tiles, so that a slot's sequence is a binary search over b and the
// number of slots, T / R + sequences + 2, is known on the host.  Rows in front
// of the first sequence and rows behind the last count as one more each,
// without tokens.  Rows without tokens get zeros.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cmath>
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) unsigned uint4v;

struct BF {
  static constexpr bool NARROW = false;  // fp32's range
  static constexpr float LIFT = 0.f;     // forward: the largest p is 2^LIFT
  static __device__ __forceinline__ float16v mfma(short8 a, short8 b,
                                                  float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
  }
  static __device__ __forceinline__ short8 pack(const float* v) {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (__bf16)v[j];
    return __builtin_bit_cast(short8, r);
  }
  static __device__ __forceinline__ short one(float v) {
    return __builtin_bit_cast(short, (__bf16)v);
  }
  static __device__ __forceinline__ float up(short v) { return bf16_to_f32(v); }
};

struct FH {
  static constexpr bool NARROW = true;   // 2^-24 to 2^16
  static constexpr float LIFT = 7.f;
  static __device__ __forceinline__ float16v mfma(short8 a, short8 b,
                                                  float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
        0);
  }
  static __device__ __forceinline__ short8 pack(const float* v) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (_Float16)v[j];
    return __builtin_bit_cast(short8, r);
  }
  static __device__ __forceinline__ short one(float v) {
    return __builtin_bit_cast(short, (_Float16)v);
  }
  static __device__ __forceinline__ float up(short v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
};

// The other half's value (lane l ^ 32).
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(
      __builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false,
      false);
  // r[0]: the low half's value in both halves, r[1]: the high half's
  return __builtin_bit_cast(float, threadIdx.x & 32 ? r[0] : r[1]);
}

// Powers of two for the operands of backward that fp16 could not hold (8192
// tokens, 16 and 4 heads of 128, training: 3-4% of the time).  p is
// about 1 / keys and dS = p (dP - D) is as much smaller than dO: unscaled,
// 2048 tokens with dO of 1e-3 lose 2% of dQ to values under 2^-24.  p <= 1 is
// held as 2^12 p.  dS goes in as g dS, a g for each accumulator's column:
// it begins as 2^30 and gives way, the accumulator with it, where a value
// passes 2^15, so that what is held reaches down to 2^-32 of the largest.
// The factors, and the scale of the scores, come off the sums in 32 bits.
constexpr float kPExp = 12.f, kPBy = 0x1p-12f;
constexpr float kStart = 0x1p30f, kMost = 0x1p15f;

// 1, or what brings the largest of a column's v to between 2^6 and 2^7 if it
// is over 2^15; both halves of a column get the same.
template <class E>
__device__ __forceinline__ float giving_way(const float (&v)[16]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[i]));
  top = fmaxf(top, other_half(top));
  return top > kMost ? __builtin_amdgcn_ldexpf(
                           1.f, min(7 - __builtin_amdgcn_frexp_expf(top), 0))
                     : 1.f;
}

// What rounding took from 8 values.
template <class E>
__device__ __forceinline__ short8 rest(const float* v, short8 rounded) {
  float w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = v[j] - E::up(rounded[j]);
  return E::pack(w);
}

constexpr int NW = 4, NTH = NW * 64;
constexpr int TILE = 64;           // rows of a staged tile
constexpr int OWN = 32 * NW;       // rows that a block owns: 32 a wave

struct Args {
  const short *q, *k, *v, *o, *dout;
  short *out, *dq, *dk, *dv;
  float *lse, *drow;               // [H, T]: -log sum exp(s) / scale, and -D
  float* part;                     // [splits][dk, dv][T, HK, D]
  const int *cu, *lengths;         // lengths may be null
  long q_t, q_h, k_t, k_h, v_t, v_h, d_t, d_h;  // strides; d: dout
  int T, B, H, HK, D, slots, splits, window;    // window 0: none
  float scale;
};

__device__ const uint4v kZeros = {0, 0, 0, 0};
__device__ const float kNoLse = -INFINITY;

// ---- which rows --------------------------------------------------------

struct Seq {
  int begin, rows, len;            // first row, all rows, tokens
};

// Where sequence i begins: 1 to B are the caller's, 0 and B + 1 the rows in
// front of them and behind them.
__device__ __forceinline__ int bound_of(const Args& a, int i) {
  return i == 0 ? 0 : i > a.B + 1 ? a.T : min(max(a.cu[i - 1], 0), a.T);
}

// The sequence and first row (in it) of a slot; false: the slot is not used.
template <int R>
__device__ __forceinline__ bool tile_of(const Args& a, int slot, Seq& s,
                                        int& row0) {
  int lo = 0, hi = a.B + 1;        // the last i whose slots begin at or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (bound_of(a, mid) / R + mid <= slot) lo = mid; else hi = mid - 1;
  }
  s.begin = bound_of(a, lo);
  s.rows = max(bound_of(a, lo + 1) - s.begin, 0);
  s.len = lo == 0 || lo > a.B ? 0 : s.rows;
  if (a.lengths && s.len) s.len = min(max(a.lengths[lo - 1], 0), s.rows);
  row0 = (slot - (s.begin / R + lo)) * R;
  return row0 >= 0 && row0 < s.rows;
}

// A product's second factor, p or dS, is rounded to the type of the first.
// Over many tokens that costs a fixed 1.4 times what rounding the results
// costs; over few it swings about that.  FINE: in a sequence of up to 256
// tokens the rest of the rounding goes through a product of its own, which
// leaves the results' own rounding, whatever else the call holds.  Forward
// and backward, without it: 256 sequences of 32 tokens, 16 and 4 heads of 64,
// 107 us (96); 40 of 200 tokens, 16 and 4 heads of 128, 196 us (182).
__device__ __forceinline__ bool is_fine(const Seq& s) { return s.len <= 256; }

// A unit is one slot of one of `heads` kv heads; its `rep` query heads are
// neighbours in time on one XCD (blocks go to the 8 XCDs in turn), so that
// they find its keys in that XCD's L2.  Heads change fastest, so that every
// XCD gets tiles of all places; `late` slots go first where those are the
// long ones.
__device__ __forceinline__ bool unit_of(const Args& a, int heads, int rep,
                                        bool late, int& head, int& slot,
                                        int& sub) {
  const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
  const int unit = j / rep * 8 + xcd;
  sub = j % rep;
  head = unit % heads;
  slot = unit / heads;
  if (slot >= a.slots) return false;
  if (late) slot = a.slots - 1 - slot;
  return true;
}

// ---- LDS tiles ---------------------------------------------------------
// A tile is [TILE][DP] with its 16-byte chunks swizzled: chunk c of row r
// stands at c ^ mix(r).  Two kinds of reads have to miss each other's banks
// (64 of 4 bytes): 16 rows at one chunk, and 4 neighbouring rows at 64
// neighbouring bytes.

template <int DP> __device__ __forceinline__ int mix(int r) {
  if constexpr (DP == 128) return (r & 3) << 2 | (r >> 2 & 3);
  return (r >> 1 & 1) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1);
}

// Every buffer is an array of its own and every tile names the ones that it
// reads and fills: only then does the compiler see that a read need not wait
// for the tile that is still on its way.

// Rows of p (stride `ld`) go to LDS without passing registers, 16 bytes a
// lane.  One offset a lane serves all of its pieces: they are NTH / NCH rows
// apart, at which the swizzle repeats, so the rest of the address is uniform.
template <int DP>
__device__ __forceinline__ unsigned stage_offset(long ld) {
  constexpr int NCH = DP / 8;
  const int r = threadIdx.x / NCH, c = (threadIdx.x % NCH) ^ mix<DP>(r);
  return (unsigned)(r * ld * 2 + c * 16);
}

__device__ __forceinline__ void to_lds(const void* src, char* tile, int it) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned*)src,
      (__attribute__((address_space(3))) unsigned*)
          (tile + (it * NTH + (threadIdx.x & ~63)) * 16),
      16, 0, 0);
}

// Rows from `rows` on and values from D on are zeros: those lanes read
// zeros instead, so nothing of another sequence ever enters a product.
template <int DP, int ROWS>
__device__ __forceinline__ void stage(const short* p, long ld, unsigned off,
                                      int row0, int rows, int D, char* tile) {
  constexpr int NCH = DP / 8, STEP = NTH / NCH;
  if (row0 + ROWS <= rows && D == DP) {
    const char* g = (const char*)(p + row0 * ld);
#pragma unroll
    for (int it = 0; it < ROWS / STEP; ++it)
      to_lds(g + it * (STEP * ld * 2) + off, tile, it);
  } else {
#pragma unroll
    for (int it = 0; it < ROWS / STEP; ++it) {
      const int r = it * STEP + threadIdx.x / NCH;
      const int c = (threadIdx.x % NCH) ^ mix<DP>(r);
      const bool ok = row0 + r < rows && c * 8 < D;
      const short* g = p + (row0 + r) * ld + c * 8;
      to_lds(ok ? (const void*)g : (const void*)&kZeros, tile, it);
    }
  }
}

// Where a lane reads in a tile.  The swizzle repeats after 16 rows, and the
// steps along a row change other bits of the chunk than the lane does: both
// kinds of reads are one offset of the lane, one XOR with a constant and a
// constant more.
template <int DP> struct Lane {
  unsigned row, col[2];

  __device__ __forceinline__ explicit Lane(int lane) {
    const int r = lane & 31;
    row = r * DP * 2 + (((lane >> 5) ^ mix<DP>(r)) << 4);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int j = lane & 15, rb = 8 * b + 4 * (lane >> 5) + (j >> 2);
      const int c = (lane >> 4 & 1) * 2 + (j >> 1 & 1);
      col[b] = rb * DP * 2 + ((c ^ mix<DP>(rb)) << 4) + (j & 1) * 8;
    }
  }
  // Forget what was worked out from the offsets: registers are dearer than
  // the XORs.
  __device__ __forceinline__ void again() {
    asm volatile("" : "+v"(row), "+v"(col[0]), "+v"(col[1]));
  }
  // A (or B) operand from rows: row r0 + l % 32, values 16 kk + 8 (l / 32)
  // + 0..7.
  __device__ __forceinline__ short8 rows(const char* tile, int r0,
                                         int kk) const {
    return *reinterpret_cast<const short8*>(tile + (row ^ kk << 5) +
                                            r0 * DP * 2);
  }
  // A operand from columns: value 32 f + l % 32 of 8 rows, in the order of
  // an accumulator: r0 + 4 (l / 32) + 0..3 and r0 + 8 + 4 (l / 32) + 0..3.
  // In a transposing read the 16 lanes of a group name 4 rows of 16 values,
  // 4 values each, and lane j of the group gets value j of the 4 rows.
  __device__ __forceinline__ short8 cols(const char* tile, int r0,
                                         int f) const {
    short4v part[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      part[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) short4v*)(
              tile + (col[b] ^ f << 6) + r0 * DP * 2));
    return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// B operand straight from global memory: row of this lane, DC / 16 steps.
template <int DC>
__device__ __forceinline__ void own_rows(const short* p, bool ok, int D,
                                         int lane, short8 (&v)[DC / 16]) {
#pragma unroll
  for (int kk = 0; kk < DC / 16; ++kk) {
    const int d = 16 * kk + 8 * (lane >> 5);
    v[kk] = ok && d < D ? *reinterpret_cast<const short8*>(p + d)
                        : short8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

// The accumulator of a [DC][32 rows] product: lane's row gets its values.
template <class E, int DC>
__device__ __forceinline__ void put_rows(short* p, bool live, int D, int lane,
                                         float by, const float16v (&acc)[DC / 32]) {
#pragma unroll
  for (int f = 0; f < DC / 32; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * f + 8 * g + 4 * (lane >> 5);
      short4v w;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = live ? E::one(acc[f][4 * g + j] * by) : (short)0;
      if (d < D) *reinterpret_cast<short4v*>(p + d) = w;
    }
}

// The order of instructions in the block of code that a call ends: so many
// LDS reads, matrix or vector instructions next.
template <int N> __device__ __forceinline__ void sched_reads() {
  __builtin_amdgcn_sched_group_barrier(0x100, N, 0);
}
template <int N> __device__ __forceinline__ void sched_mfma() {
  __builtin_amdgcn_sched_group_barrier(0x8, N, 0);
}
template <int N> __device__ __forceinline__ void sched_vector() {
  __builtin_amdgcn_sched_group_barrier(0x402, N, 0);
}
// N times: a product, READS reads, VECTOR vector instructions.
template <int N, int READS, int VECTOR>
__device__ __forceinline__ void order() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sched_mfma<1>();
    sched_reads<READS>();
    if constexpr (VECTOR > 0) sched_vector<VECTOR>();
  }
}

// 2^x; results under 2^-126 are 0
__device__ __forceinline__ float exp2_of(float x) {
  return __builtin_amdgcn_exp2f(x);
}

constexpr float kNone = -INFINITY;
constexpr float kLog2e = 1.44269504088896340736f;

// What the rows first..first + 31 of a wave see of the tile at kv0: nothing
// (0), part of it (1) or all of it (2).
template <bool CAUSAL>
__device__ __forceinline__ int sees(const Args& a, int kv0, int first,
                                    int len) {
  const int last = first + 31;
  if (first >= len || (CAUSAL && kv0 > last) ||
      (a.window && kv0 + TILE <= first - a.window + 1))
    return 0;
  return kv0 + TILE > len || (CAUSAL && kv0 + TILE - 1 > first) ||
                 (a.window && kv0 <= last - a.window)
             ? 1 : 2;
}

template <bool CAUSAL>
__device__ __forceinline__ bool seen(const Args& a, int key, int row,
                                     int len) {
  return key < len && (!CAUSAL || key <= row) &&
         (!a.window || key > row - a.window);
}

// ---- forward -----------------------------------------------------------
// DP: values of a row in LDS, DC: those that products take.

// With 128 registers, for four waves on a SIMD, heads of 64 values have their
// products in a worse order: 8192 tokens, 16 and 4 heads, causal, take 197 us,
// 175 with three waves (256 sequences of 32 tokens 31 and 36).

template <class E, int DP, int DC, bool CAUSAL>
__global__ __attribute__((amdgpu_flat_work_group_size(NTH, NTH),
                          amdgpu_waves_per_eu(2, 3))) void
packed_fwd_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) char k0[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char v0[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char k1[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char v1[TILE * DP * 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rep = a.H / a.HK;
  Lane<DP> at_lane(lane);
  int kvh, slot, sub, row0;
  Seq s;
  if (!unit_of(a, a.HK, rep, CAUSAL, kvh, slot, sub)) return;
  if (!tile_of<OWN>(a, slot, s, row0)) return;
  const int head = kvh * rep + sub;
  const int first = row0 + wave * 32, row = first + (lane & 31);
  const bool live = row < s.len;
  const long at = s.begin + row;

  // m: the reference that exponents are taken from, in units of log 2
  float m = kNone, l = 0.f;
  float16v o[DC / 32];
#pragma unroll
  for (int f = 0; f < DC / 32; ++f) o[f] = (float16v)(0.f);

  if (row0 < s.len) {
    short8 q[DC / 16];
    own_rows<DC>(a.q + at * a.q_t + head * a.q_h, live, a.D, lane, q);
    const short* kp = a.k + s.begin * a.k_t + kvh * a.k_h;
    const short* vp = a.v + s.begin * a.v_t + kvh * a.v_h;
    const unsigned koff = stage_offset<DP>(a.k_t);
    const unsigned voff = stage_offset<DP>(a.v_t);
    const int end = CAUSAL ? min(s.len, row0 + OWN) : s.len;
    const int t1 = (end + TILE - 1) / TILE;
    const float sl2 = a.scale * kLog2e;
    auto fetch = [&](int t, char* k, char* v) {
      stage<DP, TILE>(kp, a.k_t, koff, t * TILE, s.len, a.D, k);
      stage<DP, TILE>(vp, a.v_t, voff, t * TILE, s.len, a.D, v);
    };
    // One tile, while the next one is on its way to the other buffers.
    auto tile = [&](auto fine, int t, const char* kt, const char* vt, char* kn,
                    char* vn) __attribute__((always_inline)) {
      constexpr bool FINE = decltype(fine)::value;
      const int kv0 = t * TILE;
      if (t + 1 < t1) fetch(t + 1, kn, vn);
      const int what = sees<CAUSAL>(a, kv0, first, s.len);
      if (what) {
        float16v sc[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          sc[kb] = (float16v)(0.f);
#pragma unroll
          for (int kk = 0; kk < DC / 16; ++kk)
            sc[kb] = E::mfma(at_lane.rows(kt, 32 * kb, kk), q[kk], sc[kb]);
        }
        if (what == 1) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key =
                  kv0 + 32 * kb + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
              if (!seen<CAUSAL>(a, key, row, s.len)) sc[kb][i] = kNone;
            }
        }
        float top = kNone;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[kb][i]);
        top = fmaxf(top, other_half(top)) * sl2;
        // The reference moves only where a maximum leaves it by more than
        // 2^8: o and l are fp32, and probabilities keep their relative
        // precision up to there.  In fp16 the largest one stands at 2^7 to
        // 2^15 then: many keys 2^-25 below the largest are still held.
        if (__any(top > m + (8.f + E::LIFT))) {
          const float mn = fmaxf(m, top - E::LIFT);
          const float alpha = mn == kNone ? 0.f : exp2_of(m - mn);
          m = mn;
          l *= alpha;
#pragma unroll
          for (int f = 0; f < DC / 32; ++f)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[f][i] *= alpha;
        }
        const float ref = m == kNone ? 0.f : m;
        // A wave that has its probabilities goes before one that has not:
        // that keeps the two waves of a SIMD in different phases, one in
        // matrix and one in vector instructions (297 us without, 277 with,
        // 8192 tokens of 16/4 heads of 128).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          float p[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            p[j] = exp2_of(sc[ks / 2][8 * (ks & 1) + j] * sl2 - ref);
            l += p[j];
          }
          // probabilities are rounded to the type of v, which the matrix
          // product needs; their sum is taken before
          const short8 pb = E::pack(p);
          [[maybe_unused]] const short8 pr = rest<E>(p, pb);
#pragma unroll
          for (int f = 0; f < DC / 32; ++f) {
            const short8 vf = at_lane.cols(vt, 16 * ks, f);
            o[f] = E::mfma(vf, pb, o[f]);
            if constexpr (FINE) o[f] = E::mfma(vf, pr, o[f]);
          }
        }
        // the first probabilities, then a few more beside each product, whose
        // fragments are read two products ahead
        if constexpr (!FINE) {
          sched_reads<4>();
          sched_vector<36>();
          order<DC / 8 - 2, 2, 6>();
          sched_mfma<2>();
        }
        __builtin_amdgcn_s_setprio(0);
      }
      __syncthreads();
    };
    auto walk = [&](auto fine) __attribute__((always_inline)) {
      int t = a.window ? max(row0 - a.window + 1, 0) / TILE : 0;
      fetch(t, k0, v0);
      __syncthreads();
      for (; t < t1; ++t) {
        tile(fine, t, k0, v0, k1, v1);
        if (++t < t1) tile(fine, t, k1, v1, k0, v0);
      }
    };
    if (is_fine(s)) walk(std::true_type());
    else walk(std::false_type());
  }
  l += other_half(l);
  if (row < s.rows) {
    put_rows<E, DC>(a.out + (at * a.H + head) * a.D, live, a.D, lane, 1.f / l,
                    o);
    // a row without keys: exp(s - inf) is 0 in backward
    if (lane < 32)
      a.lse[(long)head * a.T + at] =
          live ? -(m + log2f(l)) / (a.scale * kLog2e) : kNone;
  }
}

// ---- backward: dQ, and D for the other kernel --------------------------

template <class E, int DP, int DC, bool CAUSAL>
__global__ __launch_bounds__(NTH, 2) void packed_bwd_q_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) char k0[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char v0[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char k1[TILE * DP * 2];
  __shared__ __attribute__((aligned(16))) char v1[TILE * DP * 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rep = a.H / a.HK;
  Lane<DP> at_lane(lane);
  int kvh, slot, sub, row0;
  Seq s;
  if (!unit_of(a, a.HK, rep, CAUSAL, kvh, slot, sub)) return;
  if (!tile_of<OWN>(a, slot, s, row0)) return;
  const int head = kvh * rep + sub;
  const int first = row0 + wave * 32, row = first + (lane & 31);
  const bool live = row < s.len;
  const long at = s.begin + row;

  float16v dq[DC / 32];
#pragma unroll
  for (int f = 0; f < DC / 32; ++f) dq[f] = (float16v)(0.f);
  float g = E::NARROW ? kStart : 1.f, drg = 0.f;  // drg: g D

  if (row0 < s.len) {
    short8 q[DC / 16], dO[DC / 16];
    own_rows<DC>(a.q + at * a.q_t + head * a.q_h, live, a.D, lane, q);
    own_rows<DC>(a.dout + at * a.d_t + head * a.d_h, live, a.D, lane, dO);
    float dr = 0.f;
    {
      short8 ov[DC / 16];
      own_rows<DC>(a.o + (at * a.H + head) * a.D, live, a.D, lane, ov);
#pragma unroll
      for (int kk = 0; kk < DC / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          dr += E::up(ov[kk][j]) * E::up(dO[kk][j]);
      dr += other_half(dr);
    }
    const float lse =
        live ? -a.lse[(long)head * a.T + at] * (a.scale * kLog2e) : INFINITY;
    const short* kp = a.k + s.begin * a.k_t + kvh * a.k_h;
    const short* vp = a.v + s.begin * a.v_t + kvh * a.v_h;
    const unsigned koff = stage_offset<DP>(a.k_t);
    const unsigned voff = stage_offset<DP>(a.v_t);
    const int end = CAUSAL ? min(s.len, row0 + OWN) : s.len;
    const int t1 = (end + TILE - 1) / TILE;
    const float sl2 = a.scale * kLog2e;
    auto fetch = [&](int t, char* k, char* v) {
      stage<DP, TILE>(kp, a.k_t, koff, t * TILE, s.len, a.D, k);
      stage<DP, TILE>(vp, a.v_t, voff, t * TILE, s.len, a.D, v);
    };
    int t = a.window ? max(row0 - a.window + 1, 0) / TILE : 0;
    // D = dO.o carries the rounding of o, and of the probabilities that went
    // into it: next to nothing where many keys share a row, but with few it
    // is half of the error of dQ and dK.  Where a block's rows see no more
    // keys than its two buffers hold, D is the sum of p dP instead (3 us more
    // for 32 rows of 128 tokens, 12 heads of 64; with sequences of 20 tokens
    // dQ and dK are off by what rounding their exact values costs, else by
    // 1.1 times that).  So it is in a narrow window, whose tiles are fetched
    // twice for it (windows of 2, 4, 8 and 32 keys in longer sequences: 1.4
    // times for 2.3, 1.8, 1.6 and 1.5; 4096 tokens, 8 and 2 heads of 64,
    // forward and backward: 51 us for 47 with a window of 8, 50 for 46 with
    // one of 64).
    const bool few = t1 - t <= 2;
    const bool narrow = a.window && a.window <= TILE;
    auto dots = [&](int t, const char* kt, const char* vt)
        __attribute__((always_inline)) {
      const int kv0 = t * TILE;
      if (!sees<CAUSAL>(a, kv0, first, s.len)) return;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        float16v sc = (float16v)(0.f), dp = (float16v)(0.f);
#pragma unroll
        for (int kk = 0; kk < DC / 16; ++kk) {
          sc = E::mfma(at_lane.rows(kt, 32 * kb, kk), q[kk], sc);
          dp = E::mfma(at_lane.rows(vt, 32 * kb, kk), dO[kk], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kv0 + 32 * kb + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
          if (seen<CAUSAL>(a, key, row, s.len))
            dr += exp2_of(sc[i] * sl2 - lse) * dp[i];
        }
      }
    };
    auto tile = [&](auto fine, int t, const char* kt, const char* vt, char* kn,
                    char* vn) __attribute__((always_inline)) {
      constexpr bool FINE = decltype(fine)::value;
      const int kv0 = t * TILE;
      if (!few && t + 1 < t1) fetch(t + 1, kn, vn);
      const int what = sees<CAUSAL>(a, kv0, first, s.len);
      if (what) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float16v sc = (float16v)(0.f), dp = (float16v)(0.f);
#pragma unroll
          for (int kk = 0; kk < DC / 16; ++kk) {
            sc = E::mfma(at_lane.rows(kt, 32 * kb, kk), q[kk], sc);
            dp = E::mfma(at_lane.rows(vt, 32 * kb, kk), dO[kk], dp);
          }
          if (what == 1) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key =
                  kv0 + 32 * kb + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
              if (!seen<CAUSAL>(a, key, row, s.len)) sc[i] = kNone;
            }
          }
          float ds[16];
          // dS is rounded to the type of k, which the product needs
#pragma unroll
          for (int i = 0; i < 16; ++i)
            ds[i] = exp2_of(sc[i] * sl2 - lse) *
                    (E::NARROW ? dp[i] * g - drg : dp[i] - drg);
          if constexpr (E::NARROW) {
            const float by = giving_way<E>(ds);
            if (__any(by < 1.f)) {
              g *= by;
              drg *= by;
#pragma unroll
              for (int i = 0; i < 16; ++i) ds[i] *= by;
#pragma unroll
              for (int f = 0; f < DC / 32; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i) dq[f][i] *= by;
            }
          }
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const short8 b = E::pack(ds + 8 * ks);
            [[maybe_unused]] const short8 r = rest<E>(ds + 8 * ks, b);
#pragma unroll
            for (int f = 0; f < DC / 32; ++f) {
              const short8 kf = at_lane.cols(kt, 32 * kb + 16 * ks, f);
              dq[f] = E::mfma(kf, b, dq[f]);
              if constexpr (FINE) dq[f] = E::mfma(kf, r, dq[f]);
            }
          }
        }
      }
      __syncthreads();
    };
    if (few || narrow) dr = 0.f;
    if (narrow && !few)
      for (int i = t; i < t1; ++i) {
        fetch(i, k0, v0);
        __syncthreads();
        dots(i, k0, v0);
        __syncthreads();
      }
    fetch(t, k0, v0);
    if (few && t + 1 < t1) fetch(t + 1, k1, v1);
    __syncthreads();
    if (few) {
      dots(t, k0, v0);
      if (t + 1 < t1) dots(t + 1, k1, v1);
    }
    if (few || narrow) dr += other_half(dr);
    if (live && lane < 32) a.drow[(long)head * a.T + at] = -dr;
    drg = dr * g;
    auto walk = [&](auto fine) __attribute__((always_inline)) {
      for (; t < t1; ++t) {
        tile(fine, t, k0, v0, k1, v1);
        if (++t < t1) tile(fine, t, k1, v1, k0, v0);
      }
    };
    if (is_fine(s)) walk(std::true_type());
    else walk(std::false_type());
  }
  if (row < s.rows)
    put_rows<E, DC>(a.dq + (at * a.H + head) * a.D, live, a.D, lane,
                    a.scale / g, dq);
}

// ---- backward: dK and dV -----------------------------------------------
// A block owns 128 keys of one kv head and goes through the query tiles of
// all its heads.  Where kv heads and key tiles are too few to fill the card,
// or to even out their lengths, the query tiles are split among blocks, which
// leave their sums in fp32, and one more kernel adds those in a fixed order.
//
// Registers are what this kernel is short of: two accumulators of 32 x DP
// and a fragment of k take 160 of the 256 that two waves on a SIMD leave, so
// v stays in LDS, query tiles are 32 rows, and LDS offsets are worked out
// again for each tile (a spilled register in this loop doubles its time).

constexpr int QT = 32;

template <class E, int DP, int DC, bool CAUSAL>
__global__ __launch_bounds__(NTH, DP == 64 ? 3 : 2) void packed_bwd_kv_kernel(
    const Args a) {
  __shared__ __attribute__((aligned(16))) char own_v[OWN * DP * 2];
  __shared__ __attribute__((aligned(16))) char q0[QT * DP * 2];
  __shared__ __attribute__((aligned(16))) char d0[QT * DP * 2];
  __shared__ __attribute__((aligned(16))) char q1[QT * DP * 2];
  __shared__ __attribute__((aligned(16))) char d1[QT * DP * 2];
  __shared__ __attribute__((aligned(16))) float s0[2 * QT];
  __shared__ __attribute__((aligned(16))) float s1[2 * QT];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rep = a.H / a.HK;
  Lane<DP> at_lane(lane);
  int vh, slot, none, row0;
  Seq s;
  if (!unit_of(a, a.HK * a.splits, 1, false, vh, slot, none)) return;
  if (!tile_of<OWN>(a, slot, s, row0)) return;
  const int kvh = vh / a.splits, split = vh % a.splits;
  const int first = row0 + wave * 32, key = first + (lane & 31);
  const bool live = key < s.len;
  const long at = s.begin + key;

  float16v dk[DC / 32], dv[DC / 32];
#pragma unroll
  for (int f = 0; f < DC / 32; ++f) dk[f] = dv[f] = (float16v)(0.f);
  float g = E::NARROW ? kStart * kPBy : 1.f;  // p brings its own factor

  if (row0 < s.len) {
    short8 k[DC / 16];
    own_rows<DC>(a.k + at * a.k_t + kvh * a.k_h, live, a.D, lane, k);
    stage<DP, OWN>(a.v + s.begin * a.v_t + kvh * a.v_h, a.v_t,
                   stage_offset<DP>(a.v_t), row0, s.len, a.D, own_v);
    const unsigned qoff = stage_offset<DP>(a.q_t);
    const unsigned doff = stage_offset<DP>(a.d_t);
    const int t0 = CAUSAL ? row0 / QT : 0;
    int end = s.len;
    if (a.window) end = min(end, row0 + OWN - 1 + a.window);
    const int t1 = (end + QT - 1) / QT;
    const int last = first + 31;
    const float sl2 = a.scale * kLog2e;
    // a query tile, its lse and its D
    auto fetch = [&](int head, int t, char* q, char* d, float* st) {
      stage<DP, QT>(a.q + s.begin * a.q_t + head * a.q_h, a.q_t, qoff, t * QT,
                    s.len, a.D, q);
      stage<DP, QT>(a.dout + s.begin * a.d_t + head * a.d_h, a.d_t, doff,
                    t * QT, s.len, a.D, d);
      if (wave == 0) {
        const int r = t * QT + (lane & 31);
        const long e = (long)head * a.T + s.begin + r;
        const float* src = lane < 32 ? a.lse + e : a.drow + e;
        if (r >= s.len) src = lane < 32 ? &kNoLse : (const float*)&kZeros;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) unsigned*)src,
            (__attribute__((address_space(3))) unsigned*)st, 4, 0, 0);
      }
    };
    // Of all query tiles of all heads this block takes its share.  From the
    // last tile down: blocks of one head begin at the same ones.
    const long tiles = t1 - t0, all = rep * tiles;
    long n = all * split / a.splits;
    const long stop = all * (split + 1) / a.splits;
    int head = kvh * rep + (int)(n / tiles), t = t1 - 1 - (int)(n % tiles);
    auto tile = [&](auto fine, const char* qt, const char* dt, const float* st,
                    char* qn, char* dn, float* sn)
        __attribute__((always_inline)) {
      constexpr bool FINE = decltype(fine)::value;
      const int r0 = t * QT;
      at_lane.again();
      if (--t < t0) {
        t = t1 - 1;
        ++head;
      }
      if (++n < stop) fetch(head, t, qn, dn, sn);
      if ((!CAUSAL || r0 + QT > first) && first < s.len &&
          (!a.window || r0 <= last + a.window - 1)) {
        float16v sc, dp;           // begin as -lse and -D of their rows
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int r = 8 * h + 4 * (lane >> 5);
          const float4v ls = *reinterpret_cast<const float4v*>(st + r);
          const float4v dr = *reinterpret_cast<const float4v*>(st + QT + r);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[4 * h + j] = ls[j];
            dp[4 * h + j] = dr[j];
          }
        }
#pragma unroll
        for (int kk = 0; kk < DC / 16; ++kk) {
          sc = E::mfma(at_lane.rows(qt, 0, kk), k[kk], sc);
          dp = E::mfma(at_lane.rows(dt, 0, kk),
                       at_lane.rows(own_v, wave * 32, kk), dp);
        }
        if ((CAUSAL && r0 < last) ||
            (a.window && r0 + QT - 1 >= first + a.window)) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int row = r0 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
            if (!seen<CAUSAL>(a, key, row, s.len)) sc[i] = kNone;
          }
        }
        float p[16], ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          p[i] = exp2_of(E::NARROW ? sc[i] * sl2 + kPExp : sc[i] * sl2);
          ds[i] = p[i] * (E::NARROW ? dp[i] * g : dp[i]);
        }
        if constexpr (E::NARROW) {
          const float by = giving_way<E>(ds);
          if (__any(by < 1.f)) {
            g *= by;
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] *= by;
#pragma unroll
            for (int f = 0; f < DC / 32; ++f)
#pragma unroll
              for (int i = 0; i < 16; ++i) dk[f][i] *= by;
          }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const short8 pb = E::pack(p + 8 * ks), sb = E::pack(ds + 8 * ks);
          [[maybe_unused]] const short8 pr = rest<E>(p + 8 * ks, pb);
          [[maybe_unused]] const short8 sr = rest<E>(ds + 8 * ks, sb);
#pragma unroll
          for (int f = 0; f < DC / 32; ++f) {
            const short8 df = at_lane.cols(dt, 16 * ks, f);
            const short8 qf = at_lane.cols(qt, 16 * ks, f);
            dv[f] = E::mfma(df, pb, dv[f]);
            dk[f] = E::mfma(qf, sb, dk[f]);
            if constexpr (FINE) {
              dv[f] = E::mfma(df, pr, dv[f]);
              dk[f] = E::mfma(qf, sr, dk[f]);
            }
          }
        }
        if constexpr (!FINE) {
          // reads stay four fragments ahead of the products
          sched_reads<8>();
          order<4 * (DC / 32) - 4, 2, 0>();
          sched_mfma<4>();
        }
      }
      __syncthreads();
    };
    if (n < stop) fetch(head, t, q0, d0, s0);
    __syncthreads();
    auto walk = [&](auto fine) __attribute__((always_inline)) {
      while (n < stop) {
        tile(fine, q0, d0, s0, q1, d1, s1);
        if (n < stop) tile(fine, q1, d1, s1, q0, d0, s0);
      }
    };
    if (is_fine(s)) walk(std::true_type());
    else walk(std::false_type());
  }
  if (key >= s.rows) return;
  const float dk_by = E::NARROW ? a.scale * kPBy / g : a.scale;
  const float dv_by = E::NARROW ? kPBy : 1.f;
  if (a.splits == 1) {
    put_rows<E, DC>(a.dk + (at * a.HK + kvh) * a.D, live, a.D, lane, dk_by,
                    dk);
    put_rows<E, DC>(a.dv + (at * a.HK + kvh) * a.D, live, a.D, lane, dv_by,
                    dv);
  } else {
    const long n = (long)a.T * a.HK * a.D;
    float* p = a.part + (2L * split * a.T + at) * a.HK * a.D + kvh * a.D;
#pragma unroll
    for (int f = 0; f < DC / 32; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * f + 8 * i + 4 * (lane >> 5);
        if (d >= a.D) continue;
        float4v x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = live ? dk[f][4 * i + j] * dk_by : 0.f;
          y[j] = live ? dv[f][4 * i + j] * dv_by : 0.f;
        }
        *reinterpret_cast<float4v*>(p + d) = x;
        *reinterpret_cast<float4v*>(p + n + d) = y;
      }
  }
}

// part [splits][2][n] -> dk and dv [n], n a multiple of 8
template <class E>
__global__ __launch_bounds__(NTH) void packed_bwd_sum_kernel(
    const float* __restrict__ part, short* __restrict__ dk,
    short* __restrict__ dv, long n, int splits) {
  const long i = ((long)blockIdx.x * NTH + threadIdx.x) * 8;
  if (i >= 2 * n) return;
  float v[8] = {};
  for (int k = 0; k < splits; ++k) {
    const float4v* p = reinterpret_cast<const float4v*>(part + 2 * k * n + i);
    const float4v x = p[0], y = p[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] += x[j];
      v[4 + j] += y[j];
    }
  }
  short* out = i < n ? dk + i : dv + (i - n);
  *reinterpret_cast<short8*>(out) = E::pack(v);
}

// ---- host --------------------------------------------------------------

}  // namespace

// Whether 16-byte reads can follow the strides of t [T, heads, D] (that of a
// dimension of one is never used).
bool attn_rows_aligned(const torch::Tensor& t) {
  return t.stride(2) == 1 &&
         (t.size(0) == 1 ||
          (t.stride(0) % 8 == 0 && t.stride(0) < (1 << 24))) &&
         (t.size(1) == 1 || t.stride(1) % 8 == 0) &&
         (size_t)t.data_ptr() % 16 == 0;
}

namespace {

Args args_of(const torch::Tensor& q, const torch::Tensor& k,
             const torch::Tensor& v, const torch::Tensor& cu,
             const c10::optional<torch::Tensor>& lengths, int64_t window,
             double scale) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3 &&
              k.sizes() == v.sizes() && k.size(0) == q.size(0) &&
              k.size(2) == q.size(2),
              "attn_packed: q [T,H,D], k and v [T,HK,D] on the GPU");
  const auto st = q.scalar_type();
  TORCH_CHECK((st == torch::kBFloat16 || st == torch::kHalf) &&
              k.scalar_type() == st && v.scalar_type() == st,
              "attn_packed: q, k and v must all be bf16 or fp16");
  TORCH_CHECK(k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0,
              "attn_packed: kv heads must divide q heads");
  TORCH_CHECK(q.size(2) % 8 == 0 && q.size(2) >= 8 && q.size(2) <= 128,
              "attn_packed: D must be a multiple of 8, at most 128");
  TORCH_CHECK(attn_rows_aligned(q) && attn_rows_aligned(k) && attn_rows_aligned(v),
              "attn_packed: rows must be dense and 16-byte aligned");
  TORCH_CHECK(scale > 1e-30 && scale < 1e30, "attn_packed: scale must be positive");
  TORCH_CHECK(q.size(0) < (1L << 29), "attn_packed: too many rows");
  TORCH_CHECK(cu.dim() == 1 && cu.size(0) >= 2 && cu.is_contiguous() &&
              cu.scalar_type() == torch::kInt,
              "attn_packed: cu_seqlens must be int32 [sequences + 1]");
  for (const auto& x : {k, v, cu})
    TORCH_CHECK(x.device() == q.device(),
                "attn_packed: all tensors must be on one device");
  if (lengths.has_value())
    TORCH_CHECK(lengths->dim() == 1 && lengths->size(0) == cu.size(0) - 1 &&
                lengths->is_contiguous() &&
                lengths->scalar_type() == torch::kInt &&
                lengths->device() == q.device(),
                "attn_packed: lengths must be int32 [sequences]");
  Args a = {};
  a.q = (const short*)q.data_ptr();
  a.k = (const short*)k.data_ptr();
  a.v = (const short*)v.data_ptr();
  a.q_t = q.stride(0); a.q_h = q.stride(1);
  a.k_t = k.stride(0); a.k_h = k.stride(1);
  a.v_t = v.stride(0); a.v_h = v.stride(1);
  a.cu = cu.data_ptr<int>();
  a.lengths = lengths ? lengths->data_ptr<int>() : nullptr;
  a.T = (int)q.size(0);
  a.B = (int)cu.size(0) - 1;
  a.H = (int)q.size(1);
  a.HK = (int)k.size(1);
  a.D = (int)q.size(2);
  a.window = (int)std::min<int64_t>(window, a.T);
  a.scale = (float)scale;
  const long slots = (long)a.T / OWN + a.B + 2;
  // a launch has less than 2^32 threads; heads are rounded up to 8 units
  TORCH_CHECK((slots + 8) * a.H * NTH < (1L << 32),
              "attn_packed: too many rows, sequences and heads: (rows / 128 + "
              "sequences + 10) * heads must be less than 2^24");
  a.slots = (int)slots;
  a.splits = 1;
  return a;
}

// Rows stand in LDS as 64 or 128 values; of 128, only 96 are computed with
// where D is no more (8192 tokens, 16 and 4 heads of 80, causal: 262 us
// forward and 1032 with gradients, with all 128 288 and 1184).
#define PACKED_LAUNCH(KERNEL, HEADS, REP)                                   \
  do {                                                                      \
    const dim3 grid((a.slots * (HEADS) + 7) / 8 * 8 * (REP));               \
    auto launch = [&](auto kernel) {                                        \
      hipLaunchKernelGGL(kernel, grid, dim3(NTH), 0, stream.stream(), a);   \
    };                                                                      \
    auto typed = [&](auto type) {                                           \
      using E = decltype(type);                                             \
      if (a.D <= 64 && causal) launch(KERNEL<E, 64, 64, true>);             \
      else if (a.D <= 64) launch(KERNEL<E, 64, 64, false>);                 \
      else if (a.D <= 96 && causal) launch(KERNEL<E, 128, 96, true>);       \
      else if (a.D <= 96) launch(KERNEL<E, 128, 96, false>);                \
      else if (causal) launch(KERNEL<E, 128, 128, true>);                   \
      else launch(KERNEL<E, 128, 128, false>);                              \
    };                                                                      \
    if (bf) typed(BF());                                                    \
    else typed(FH());                                                       \
  } while (0)

}  // namespace

// {o [T,H,D], lse [H,T]: -log sum exp(s) / scale, -inf for rows without tokens}
std::vector<torch::Tensor> attn_packed_fwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cu,
    c10::optional<torch::Tensor> lengths, bool causal, int64_t window,
    double scale) {
  Args a = args_of(q, k, v, cu, lengths, window, scale);
  TORCH_CHECK(window >= 0 && (window == 0 || causal),
              "attn_packed: a window needs a causal mask");
  const c10::cuda::CUDAGuard guard(q.device());
  auto o = torch::empty(q.sizes(), q.options());
  auto lse = torch::empty({a.H, a.T}, q.options().dtype(torch::kFloat32));
  if (a.T == 0) return {o, lse};
  a.out = (short*)o.data_ptr();
  a.lse = lse.data_ptr<float>();
  auto stream = c10::cuda::getCurrentCUDAStream();
  const bool bf = q.scalar_type() == torch::kBFloat16;
  PACKED_LAUNCH(packed_fwd_kernel, a.HK, a.H / a.HK);
  HIP_CHECK_LAST();
  return {o, lse};
}

// {dq, dk, dv}, contiguous
std::vector<torch::Tensor> attn_packed_bwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor o,
    torch::Tensor dout, torch::Tensor lse, torch::Tensor cu,
    c10::optional<torch::Tensor> lengths, bool causal, int64_t window,
    double scale) {
  Args a = args_of(q, k, v, cu, lengths, window, scale);
  TORCH_CHECK(dout.sizes() == q.sizes() && o.sizes() == q.sizes() &&
              o.is_contiguous() && dout.scalar_type() == q.scalar_type() &&
              o.scalar_type() == q.scalar_type() && attn_rows_aligned(dout) &&
              dout.device() == q.device(),
              "attn_packed: o and dout must be like q, dout's rows dense and "
              "16-byte aligned");
  const c10::cuda::CUDAGuard guard(q.device());
  auto dq = torch::empty(q.sizes(), q.options());
  auto dk = torch::empty(k.sizes(), k.options());
  auto dv = torch::empty(v.sizes(), v.options());
  if (a.T == 0) return {dq, dk, dv};
  auto drow = torch::empty_like(lse);
  a.o = (const short*)o.data_ptr();
  a.dout = (const short*)dout.data_ptr();
  a.d_t = dout.stride(0);
  a.d_h = dout.stride(1);
  a.dq = (short*)dq.data_ptr();
  a.dk = (short*)dk.data_ptr();
  a.dv = (short*)dv.data_ptr();
  a.lse = lse.data_ptr<float>();
  a.drow = drow.data_ptr<float>();
  auto stream = c10::cuda::getCurrentCUDAStream();
  const bool bf = q.scalar_type() == torch::kBFloat16;
  PACKED_LAUNCH(packed_bwd_q_kernel, a.HK, a.H / a.HK);
  // Two blocks of four waves on each of 256 CUs run at once: about twice as
  // many even out their lengths, but a block should keep eight query tiles
  // (of sequences of the mean length).  One document of 8192 tokens, 16 and
  // 4 heads of 128: 1656 us for the backward pass unsplit (260 blocks), 1113
  // in two, 934 in four; documents of 900 tokens, 32 and 8 heads: 711 unsplit
  // (592 blocks), 528 in two, 568 in four.
  const long units = (long)a.slots * a.HK;
  long seen = a.T / a.B + 1;
  if (a.window) seen = std::min<long>(seen, a.window + OWN);
  const long most = std::max<long>(1, seen / QT * (a.H / a.HK) / 8);
  a.splits = (int)std::min({(1023 + units) / units, most, 16L});
  torch::Tensor part;
  if (a.splits > 1) {
    part = torch::empty({a.splits, 2, a.T, a.HK, a.D}, lse.options());
    a.part = part.data_ptr<float>();
  }
  PACKED_LAUNCH(packed_bwd_kv_kernel, a.HK * a.splits, 1);
  if (a.splits > 1) {
    const long n = (long)a.T * a.HK * a.D;
    const dim3 grid((unsigned)((2 * n / 8 + NTH - 1) / NTH));
    if (bf)
      hipLaunchKernelGGL((packed_bwd_sum_kernel<BF>), grid, dim3(NTH), 0,
                         stream.stream(), a.part, a.dk, a.dv, n, a.splits);
    else
      hipLaunchKernelGGL((packed_bwd_sum_kernel<FH>), grid, dim3(NTH), 0,
                         stream.stream(), a.part, a.dk, a.dv, n, a.splits);
  }
  HIP_CHECK_LAST();
  return {dq, dk, dv};
}
