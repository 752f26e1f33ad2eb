// The junction of two residual blocks in one pass each way:
//
//   z = h r1 w1,  r1 = rsqrt(mean h^2 + eps)      norm after the block
//   s = alpha x + g z                             gate, residual scale, sum
//   n = s r2 w2,  r2 = rsqrt(mean s^2 + eps)      norm before the next
//
// and, from dn and ds (the gradients of n and s), with hh = h r1, sh = s r2:
//
//   e  = ds + r2 (dn w2 - sh mean(dn w2 sh))      all that reaches s
//   dx = alpha e,  dw2 = sum dn sh
//   u  = g e w1,   dh = r1 (u - hh mean(u hh))
//   dg = w1 sum(e hh) over the rows of one gate,  dw1 = sum g e hh
//
// Bound by memory: forward reads h, x and writes n, s; backward reads h, x,
// dn, ds and writes dh, dx (s is computed again in registers, so that it is
// neither kept nor rounded).  A row stays in the registers of its threads
// from load to store; sums are fp32.  Column sums go through one partial row
// for each block, which a second kernel adds in a fixed order.  16384 rows
// of 4096 bf16: 95 us forward, 170 + 7 us backward, 5.7 and 4.7 TB/s.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <algorithm>
#include "common.h"

namespace {

template <class T> __device__ __forceinline__ float up(T v) { return (float)v; }
template <> __device__ __forceinline__ float up(short v) {
  return bf16_to_f32(v);
}
template <class T> __device__ __forceinline__ T down(float f) { return (T)f; }
template <> __device__ __forceinline__ short down(float f) {
  return __builtin_bit_cast(short, (__bf16)f);  // one instruction for two
}

template <class T> constexpr int WIDE = 16 / sizeof(T);

typedef __attribute__((ext_vector_type(4))) unsigned uint4v;

// 16 bytes at any alignment of their own type: rows of an odd width begin
// anywhere, and global loads need no alignment beyond that
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Run {
  uint4v w;
};

// Value j of a run: 16-bit ones stand two to a register until they are used.
template <class T> __device__ __forceinline__ float part_of(uint4v w, int j) {
  if constexpr (std::is_same_v<T, float>) {
    const unsigned u = w[j];
    return __builtin_bit_cast(float, u);
  } else {
    const unsigned u = w[j / 2];
    if constexpr (std::is_same_v<T, short>)
      return __builtin_bit_cast(float, j & 1 ? u & 0xffff0000u : u << 16);
    else
      return (float)__builtin_bit_cast(
          _Float16, (unsigned short)(j & 1 ? u >> 16 : u));
  }
}

// w without its first `bytes` (1 to 15), zeros at its end.
__device__ __forceinline__ uint4v shifted(uint4v w, int bytes) {
  unsigned long lo = (unsigned long)w[1] << 32 | w[0];
  unsigned long hi = (unsigned long)w[3] << 32 | w[2];
  const int s = bytes * 8;
  lo = s < 64 ? lo >> s | hi << (64 - s) : hi >> (s - 64);
  hi = s < 64 ? hi >> s : 0;
  return uint4v{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi,
                (unsigned)(hi >> 32)};
}

template <class T> __device__ __forceinline__ unsigned bits_of(T v) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(unsigned, v);
  else return __builtin_bit_cast(unsigned short, v);
}

// w with v put before its first value.
template <class T> __device__ __forceinline__ uint4v pushed(uint4v w, T v) {
  if constexpr (sizeof(T) == 4) return uint4v{bits_of(v), w[0], w[1], w[2]};
  else return uint4v{w[0] << 16 | bits_of(v), w[1] << 16 | w[0] >> 16,
                     w[2] << 16 | w[1] >> 16, w[3] << 16 | w[2] >> 16};
}

// Writes the first n values of w (n less than a run's).
template <class T>
__device__ __forceinline__ void store_part(T* p, uint4v w, int n) {
  struct __attribute__((packed, aligned(sizeof(T)))) Two { unsigned a, b; };
  struct __attribute__((packed, aligned(sizeof(T)))) One { unsigned a; };
  constexpr int PER = 4 / sizeof(T);       // values of a register
  if (n & 2 * PER) {
    *reinterpret_cast<Two*>(p) = Two{w[0], w[1]};
    p += 2 * PER;
    w[0] = w[2];
    w[1] = w[3];
  }
  if (n & PER) {
    *reinterpret_cast<One*>(p) = One{w[0]};
    p += PER;
    w[0] = w[1];
  }
  if constexpr (PER == 2) {
    const unsigned short last = (unsigned short)w[0];
    if (n & 1) *p = __builtin_bit_cast(T, last);
  }
}

// The part of a row that a thread holds: E values as runs of 16 bytes, ROWT
// threads side by side, kept as they were read until they are used.  EVEN:
// D is a multiple of a run, so that no run ends inside of it.  Without the
// code for that, 16384 rows of 4096 bf16 take 95 and 170 us forward and
// backward; with it 102 and 176.  Rows whose width is odd begin off the lines
// of memory, too: 12474 rows of 1440 fp16 take 24 us forward, of 1435 40.
template <class T, int ROWT, int E, bool EVEN> struct Row {
  static constexpr int V = WIDE<T>, C = E / V;
  uint4v r[C];

  static __device__ __forceinline__ int at(int t, int c) {
    return (c * ROWT + t) * V;
  }
  __device__ __forceinline__ void load(const T* p, int D, int t) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = at(t, c);
      if (EVEN) {
        r[c] = (uint4v)(0);
        if (i < D) r[c] = reinterpret_cast<const Run<T>*>(p + i)->w;
      } else if (i + V <= D) {
        r[c] = reinterpret_cast<const Run<T>*>(p + i)->w;
      } else {
        r[c] = (uint4v)(0);
        if (i < D && D >= V)       // the row's last run, less what is not ours
          r[c] = shifted(reinterpret_cast<const Run<T>*>(p + D - V)->w,
                         (i + V - D) * (int)sizeof(T));
        else if (i < D)
          for (int j = D - i - 1; j >= 0; --j)
            r[c] = pushed<T>(r[c], p[i + j]);
      }
    }
  }
  __device__ __forceinline__ void ones() {
    const unsigned b = bits_of(down<T>(1.f));
#pragma unroll
    for (int c = 0; c < C; ++c)
      r[c] = (uint4v)(sizeof(T) == 2 ? b << 16 | b : b);
  }
  __device__ __forceinline__ float operator[](int i) const {
    return part_of<T>(r[i / V], i % V);
  }
  static __device__ __forceinline__ void store(T* p, int D, int t,
                                               const float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = at(t, c);
      constexpr int PER = 4 / sizeof(T);
      Run<T> w = {(uint4v)(0)};
#pragma unroll
      for (int j = 0; j < V; ++j)
        w.w[j / PER] |= bits_of(down<T>(v[c * V + j])) << (j % PER * 16);
      if (EVEN ? i < D : i + V <= D)
        *reinterpret_cast<Run<T>*>(p + i) = w;
      else if (!EVEN && i < D)
        store_part(p + i, w.w, D - i);
    }
  }
  static __device__ __forceinline__ void store32(float* p, int D, int t,
                                                 const float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (EVEN && at(t, c) >= D) continue;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (EVEN || at(t, c) + j < D) p[at(t, c) + j] = v[c * V + j];
    }
  }
};

// Sum over the ROWT threads of a row.  Two rows of scratch in turn, so that
// one barrier for each sum is enough.
template <int ROWT>
__device__ __forceinline__ float row_sum(float v, float (*scratch)[16],
                                         int& turn) {
  v = wave_reduce_sum(v);
  if constexpr (ROWT == WAVE) return v;
  const int w = threadIdx.x / WAVE;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) scratch[turn][w] = v;
  __syncthreads();
  v = scratch[turn][0];
#pragma unroll
  for (int i = 1; i < ROWT / WAVE; ++i) v += scratch[turn][i];
  return v;
}

// Rows of one wave stand four to a block; wider ones have a block each, as
// their barriers need.
template <int ROWT> constexpr int BLOCK = ROWT == WAVE ? 256 : ROWT;

// Which of the block's rows is this thread's: the same for a whole wave, and
// the compiler is told so (rows are then addressed from scalar registers).
template <int ROWT> __device__ __forceinline__ int worker_of() {
  return BLOCK<ROWT> == ROWT
             ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / ROWT);
}

// Row i uses row i / group of the gate (no gate: 1).  The next row is on its
// way while a row is worked on.
template <class T, int ROWT, int E, bool EVEN>
__global__ __launch_bounds__(BLOCK<ROWT>) void block_norm_fwd_kernel(
    const T* __restrict__ h, const T* __restrict__ x,
    const T* __restrict__ w1, const T* __restrict__ w2,
    const T* __restrict__ gate, T* __restrict__ n_out, T* __restrict__ s_out,
    float* __restrict__ r1_out, float* __restrict__ r2_out, long rows,
    long group, int D, float alpha, float eps) {
  using R = Row<T, ROWT, E, EVEN>;
  __shared__ float scratch[2][16];
  constexpr int RPB = BLOCK<ROWT> / ROWT;
  const int t = threadIdx.x % ROWT;
  const long step = (long)gridDim.x * RPB;
  long row = (long)blockIdx.x * RPB + worker_of<ROWT>();
  int turn = 0;
  R wa, wb, hr, xr, g;
  if (row < rows) {
    hr.load(h + row * D, D, t);
    xr.load(x + row * D, D, t);
  }
  wa.load(w1, D, t);
  wb.load(w2, D, t);
  g.ones();
  for (; row < rows; row += step) {
    float a[E], b[E];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      a[i] = hr[i];
      b[i] = alpha * xr[i];
      q += a[i] * a[i];
    }
    if (gate) g.load(gate + row / group * D, D, t);
    if (row + step < rows) {
      hr.load(h + (row + step) * D, D, t);
      xr.load(x + (row + step) * D, D, t);
    }
    const float r1 = rsqrtf(row_sum<ROWT>(q, scratch, turn) / D + eps);
    q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      b[i] += g[i] * (a[i] * r1 * wa[i]);
      q += b[i] * b[i];
    }
    R::store(s_out + row * D, D, t, b);
    const float r2 = rsqrtf(row_sum<ROWT>(q, scratch, turn) / D + eps);
#pragma unroll
    for (int i = 0; i < E; ++i) b[i] *= r2 * wb[i];
    R::store(n_out + row * D, D, t, b);
    if (t == 0 && r1_out) {
      r1_out[row] = r1;
      r2_out[row] = r2;
    }
  }
}

// Adds the workers of a block up: worker 0 has the sums afterwards.
template <int ROWT, int E>
__device__ __forceinline__ void block_add(float (&v)[E], float* room) {
  constexpr int RPB = BLOCK<ROWT> / ROWT;
  if constexpr (RPB > 1) {
    const int t = threadIdx.x % ROWT, w = worker_of<ROWT>();
    __syncthreads();
    if (w)
#pragma unroll
      for (int i = 0; i < E; ++i) room[((w - 1) * E + i) * ROWT + t] = v[i];
    __syncthreads();
    if (w == 0)
#pragma unroll
      for (int k = 0; k < RPB - 1; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] += room[(k * E + i) * ROWT + t];
  }
}

// Waves on a SIMD that the backward kernel leaves registers for (512 / waves).
// 16-bit rows fit 128 but for a few; of an odd width and with whole groups
// they need three waves' (12474 rows of 1001 bf16, a gate for each, forward
// and backward: 117 us, 134 with four waves, where 35 registers spill), and
// so do 32-bit rows (1024 fp32: 144 us for 169).  Blocks of 512 threads have
// 128 registers or 256: 32-bit rows take 256 (4096 rows of 4096 fp32, a gate
// for each: 173 us, 227 with 128, where up to 47 spill), 16-bit ones keep
// 128, though 37 spill at an odd width with whole groups: with 256, 4000 rows
// of 4001 and a gate for each take 151 us for 175, but 700 groups of 10 rows
// 307 for 278.  Blocks of 1024 threads have no more than 128: 13 to 68
// spill with 8 values a thread, and 136 to 504 with 16.
template <class T, int ROWT, bool EVEN, bool WHOLE>
constexpr int BWD_WAVES =
    sizeof(T) == 4 ? (ROWT > 512 ? 4 : ROWT > 256 ? 2 : 3)
                   : (ROWT <= 256 && !EVEN && WHOLE ? 3 : 4);

// A block's workers (a worker: the ROWT threads of a row) leave one partial
// row of each sum.  WHOLE: a worker takes `per` rows that are whole groups,
// and finishes their rows of dg.  Otherwise `slices` blocks share a group of
// rows, `per` rows each, which the workers take in turn, and sum(e hh) of
// the group is left in parts too.
template <class T, int ROWT, int E, bool EVEN, bool WHOLE>
__global__
__launch_bounds__(BLOCK<ROWT>, (BWD_WAVES<T, ROWT, EVEN, WHOLE>))
void block_norm_bwd_kernel(
    const T* __restrict__ dn, const T* __restrict__ ds,
    const T* __restrict__ h, const T* __restrict__ x,
    const T* __restrict__ w1, const T* __restrict__ w2,
    const T* __restrict__ gate, const float* __restrict__ r1s,
    const float* __restrict__ r2s, T* __restrict__ dh, T* __restrict__ dx,
    T* __restrict__ dg, float* __restrict__ part1, float* __restrict__ part2,
    float* __restrict__ partg, long rows, long group, long per, long slices,
    int D, float alpha) {
  using R = Row<T, ROWT, E, EVEN>;
  constexpr int RPB = BLOCK<ROWT> / ROWT;
  __shared__ float scratch[2][16];
  __shared__ float room[RPB > 1 ? (RPB - 1) * E * ROWT : 1];
  const int t = threadIdx.x % ROWT, w = worker_of<ROWT>();
  int turn = 0;
  long row, end, step;
  if (WHOLE) {
    row = ((long)blockIdx.x * RPB + w) * per;
    end = min(row + per, rows);
    step = 1;
  } else {
    const long k = blockIdx.x / slices, lo = blockIdx.x % slices * per;
    row = k * group + lo + w;
    end = k * group + min(lo + per, group);
    step = RPB;
  }
  R wa, wb, g, hr, xr, dr, er;
  float r1n, r2n;
  auto fetch = [&](long i) {
    r1n = r1s[i];
    r2n = r2s[i];
    hr.load(h + i * D, D, t);
    xr.load(x + i * D, D, t);
    dr.load(dn + i * D, D, t);
    er.load(ds + i * D, D, t);
  };
  if (row < end) fetch(row);
  wa.load(w1, D, t);
  wb.load(w2, D, t);
  g.ones();
  if (gate && !WHOLE) g.load(gate + blockIdx.x / slices * D, D, t);
  float acc1[E], acc2[E], accg[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc1[i] = acc2[i] = accg[i] = 0.f;
  for (; row < end; row += step) {
    const float r1 = r1n, r2 = r2n;
    if (gate && WHOLE) g.load(gate + row / group * D, D, t);
    float a[E], b[E], d[E], e[E];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      a[i] = hr[i] * r1;           // hh
      b[i] = (alpha * xr[i] + g[i] * (a[i] * wa[i])) * r2;  // sh
      acc2[i] += dr[i] * b[i];
      d[i] = dr[i] * wb[i];
      e[i] = er[i];
      q += d[i] * b[i];
    }
    if (row + step < end) fetch(row + step);
    q = row_sum<ROWT>(q, scratch, turn) / D;
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      e[i] += r2 * (d[i] - b[i] * q);
      b[i] = alpha * e[i];
      accg[i] += e[i] * a[i];
      d[i] = g[i] * e[i] * wa[i];  // u
      p += d[i] * a[i];
    }
    R::store(dx + row * D, D, t, b);
    p = row_sum<ROWT>(p, scratch, turn) / D;
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] = r1 * (d[i] - a[i] * p);
    R::store(dh + row * D, D, t, d);
    if (WHOLE && gate && (row + 1) % group == 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        d[i] = wa[i] * accg[i];
        acc1[i] += g[i] * accg[i];
        accg[i] = 0.f;
      }
      R::store(dg + row / group * D, D, t, d);
    }
  }
  block_add<ROWT>(acc2, room);
  if (WHOLE && gate) {
    block_add<ROWT>(acc1, room);
  } else {
    block_add<ROWT>(accg, room);
#pragma unroll
    for (int i = 0; i < E; ++i) acc1[i] = g[i] * accg[i];
  }
  if (w) return;
  R::store32(part1 + (long)blockIdx.x * D, D, t, acc1);
  R::store32(part2 + (long)blockIdx.x * D, D, t, acc2);
  if (gate && !WHOLE) R::store32(partg + (long)blockIdx.x * D, D, t, accg);
}

// blockIdx.y 0: dw1, 1: dw2, 2 + k: dg of group k, times w1.
template <class T>
__global__ __launch_bounds__(1024) void block_norm_sum_kernel(
    const float* __restrict__ part1, const float* __restrict__ part2,
    const float* __restrict__ partg, const T* __restrict__ w1,
    T* __restrict__ dw1, T* __restrict__ dw2, T* __restrict__ dg, long parts,
    long slices, int D) {
  __shared__ float sh[32][33];
  const int cl = threadIdx.x & 31, pl = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + cl;
  const long k = (long)blockIdx.y - 2;
  const float* p = k < 0 ? (blockIdx.y ? part2 : part1) : partg + k * slices * D;
  const long n = k < 0 ? parts : slices;
  float s = 0.f;
  if (i < D) {
    long r = pl;
    for (; r + 7 * 32 < n; r += 8 * 32) {  // eight loads on their way
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = p[(r + j * 32) * D + i];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; r < n; r += 32) s += p[r * D + i];
  }
  sh[pl][cl] = s;
  __syncthreads();
  // 32 row lanes of each column, now side by side in a half wave
  s = sh[cl][pl];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor(s, off, WAVE);
  const int c = blockIdx.x * 32 + pl;
  if (cl != 0 || c >= D) return;
  if (k >= 0) dg[k * D + c] = down<T>(s * up(w1[c]));
  else (blockIdx.y ? dw2 : dw1)[c] = down<T>(s);
}

struct Shape {
  long rows, group;
  int D;
};

Shape check(const torch::Tensor& h, const torch::Tensor& x,
            const torch::Tensor& w1, const torch::Tensor& w2,
            const c10::optional<torch::Tensor>& gate) {
  const auto st = h.scalar_type();
  TORCH_CHECK(h.is_cuda() && h.dim() >= 1 && h.is_contiguous() &&
              x.is_contiguous() && x.sizes() == h.sizes(),
              "block_norm: h and x must be contiguous GPU tensors of one shape");
  TORCH_CHECK(st == torch::kBFloat16 || st == torch::kHalf ||
              st == torch::kFloat32, "block_norm: bf16, fp16 or fp32 only");
  Shape s;
  s.D = (int)h.size(-1);
  TORCH_CHECK(h.size(-1) >= 1 && h.size(-1) <= 16384,
              "block_norm: the last dimension must be 1 to 16384, got ",
              h.size(-1));
  s.rows = h.numel() / s.D;
  s.group = std::max<long>(s.rows, 1);
  std::vector<torch::Tensor> others = {x, w1, w2};
  for (const auto& w : {w1, w2})
    TORCH_CHECK(w.is_contiguous() && w.dim() == 1 && w.size(0) == s.D,
                "block_norm: weights must be contiguous [D]");
  if (gate.has_value()) {
    const auto& g = *gate;
    TORCH_CHECK(g.is_contiguous() && g.dim() == 2 && g.size(1) == s.D &&
                (s.rows == 0 || (g.size(0) >= 1 && s.rows % g.size(0) == 0)),
                "block_norm: the gate must be contiguous [G, D], G a divisor "
                "of the rows");
    if (s.rows) s.group = s.rows / g.size(0);
    others.push_back(g);
  }
  for (const auto& o : others)
    TORCH_CHECK(o.scalar_type() == st && o.device() == h.device(),
                "block_norm: all tensors must have h's type and device");
  return s;
}

// Threads of a row: 8 values each, so that a row and the next one, its
// weights and its sums stay in 128 registers; wider rows need 16.
#define BY_WIDTH(T, D, ...)                                                  \
  if ((D) <= 64 * 8) { constexpr int ROWT = 64, E = 8; __VA_ARGS__; }        \
  else if ((D) <= 128 * 8) { constexpr int ROWT = 128, E = 8; __VA_ARGS__; } \
  else if ((D) <= 256 * 8) { constexpr int ROWT = 256, E = 8; __VA_ARGS__; } \
  else if ((D) <= 512 * 8) { constexpr int ROWT = 512, E = 8; __VA_ARGS__; } \
  else if ((D) <= 1024 * 8) { constexpr int ROWT = 1024, E = 8; __VA_ARGS__; } \
  else { constexpr int ROWT = 1024, E = 16; __VA_ARGS__; }

#define BY_TYPE(st, ...)                                                \
  if ((st) == torch::kBFloat16) { using T = short; __VA_ARGS__; }       \
  else if ((st) == torch::kHalf) { using T = _Float16; __VA_ARGS__; }   \
  else { using T = float; __VA_ARGS__; }

}  // namespace

// {n, s, r1, r2}; r1 and r2 are empty unless `train`.
std::vector<torch::Tensor> block_norm_fwd(torch::Tensor h, torch::Tensor x,
                                          torch::Tensor w1, torch::Tensor w2,
                                          c10::optional<torch::Tensor> gate,
                                          double alpha, double eps,
                                          bool train) {
  const Shape s = check(h, x, w1, w2, gate);
  const c10::cuda::CUDAGuard guard(h.device());
  auto n = torch::empty_like(h);
  auto sum = torch::empty_like(h);
  auto r = torch::empty({2, train ? s.rows : 0},
                        h.options().dtype(torch::kFloat32));
  auto r1 = r.select(0, 0), r2 = r.select(0, 1);
  if (s.rows == 0) return {n, sum, r1, r2};
  auto stream = c10::cuda::getCurrentCUDAStream();
  BY_TYPE(h.scalar_type(), BY_WIDTH(T, s.D, {
    constexpr int RPB = BLOCK<ROWT> / ROWT;
    const int grid = (int)std::min<long>((s.rows + RPB - 1) / RPB,
                                         2048 * 256 / BLOCK<ROWT>);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(
          kernel, dim3(grid), dim3(BLOCK<ROWT>), 0, stream.stream(),
          (const T*)h.data_ptr(), (const T*)x.data_ptr(),
          (const T*)w1.data_ptr(), (const T*)w2.data_ptr(),
          gate ? (const T*)gate->data_ptr() : nullptr, (T*)n.data_ptr(),
          (T*)sum.data_ptr(), train ? r1.data_ptr<float>() : nullptr,
          train ? r2.data_ptr<float>() : nullptr, s.rows, s.group, s.D,
          (float)alpha, (float)eps);
    };
    if (s.D % WIDE<T> == 0) launch(block_norm_fwd_kernel<T, ROWT, E, true>);
    else launch(block_norm_fwd_kernel<T, ROWT, E, false>);
  }))
  HIP_CHECK_LAST();
  return {n, sum, r1, r2};
}

// {dh, dx, dw1, dw2, dgate (empty without a gate)}
std::vector<torch::Tensor> block_norm_bwd(
    torch::Tensor dn, torch::Tensor ds, torch::Tensor h, torch::Tensor x,
    torch::Tensor w1, torch::Tensor w2, c10::optional<torch::Tensor> gate,
    torch::Tensor r1, torch::Tensor r2, double alpha) {
  const Shape s = check(h, x, w1, w2, gate);
  for (const auto& g : {dn, ds})
    TORCH_CHECK(g.is_contiguous() && g.sizes() == h.sizes() &&
                g.scalar_type() == h.scalar_type() &&
                g.device() == h.device(),
                "block_norm: gradients must be laid out as h");
  const c10::cuda::CUDAGuard guard(h.device());
  auto dh = torch::empty_like(h);
  auto dx = torch::empty_like(h);
  auto dw1 = torch::empty_like(w1);
  auto dw2 = torch::empty_like(w2);
  auto dg = gate ? torch::empty_like(*gate) : torch::empty({0}, h.options());
  if (s.rows == 0) return {dh, dx, dw1.zero_(), dw2.zero_(), dg.zero_()};
  auto stream = c10::cuda::getCurrentCUDAStream();
  const long groups = s.rows / s.group;
  // About 1024 blocks of 256 threads fill the card, and each adds a partial
  // row of each sum: with two rows for each worker at least, those stay
  // small beside the rows.  A group of rows is cut into as many slices as
  // that allows; where there are more groups, a worker takes several.  A
  // block of one worker takes whole groups also where they are not cut, so
  // that their rows of dg need no second kernel (1100 groups of 30 rows of
  // 1024 bf16, forward and backward: 150 us, 226 through that kernel).
  // Blocks of four workers rather share a group until there is one for each
  // block (1000 groups of 100 rows of 256: 135 us, 229 with whole ones).
  BY_TYPE(h.scalar_type(), BY_WIDTH(T, s.D, {
    constexpr int RPB = BLOCK<ROWT> / ROWT;
    const long want = std::max<long>(
        1, std::min<long>(s.rows / (2 * RPB), 1024L * 256 / BLOCK<ROWT>));
    const bool whole = (RPB > 1 ? groups : 2 * groups) > want;
    long per = 0;
    long slices = 1;
    long grid = 0;
    if (whole) {
      per = (groups + want * RPB - 1) / (want * RPB) * s.group;
      grid = (s.rows + per * RPB - 1) / (per * RPB);
    } else {
      slices = std::max<long>(1, want / groups);
      per = (s.group + slices - 1) / slices;
      slices = (s.group + per - 1) / per;
      grid = groups * slices;
    }
    auto part = torch::empty({gate && !whole ? 3 : 2, grid, s.D},
                             h.options().dtype(torch::kFloat32));
    float* p1 = part.data_ptr<float>();
    float* p2 = p1 + grid * s.D;
    float* pg = gate && !whole ? p2 + grid * s.D : nullptr;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(
          kernel, dim3((unsigned)grid), dim3(BLOCK<ROWT>), 0,
          stream.stream(), (const T*)dn.data_ptr(), (const T*)ds.data_ptr(),
          (const T*)h.data_ptr(), (const T*)x.data_ptr(),
          (const T*)w1.data_ptr(), (const T*)w2.data_ptr(),
          gate ? (const T*)gate->data_ptr() : nullptr, r1.data_ptr<float>(),
          r2.data_ptr<float>(), (T*)dh.data_ptr(), (T*)dx.data_ptr(),
          (T*)dg.data_ptr(), p1, p2, pg, s.rows, s.group, per, slices, s.D,
          (float)alpha);
    };
    if (s.D % WIDE<T> == 0) {
      if (whole) launch(block_norm_bwd_kernel<T, ROWT, E, true, true>);
      else launch(block_norm_bwd_kernel<T, ROWT, E, true, false>);
    } else {
      if (whole) launch(block_norm_bwd_kernel<T, ROWT, E, false, true>);
      else launch(block_norm_bwd_kernel<T, ROWT, E, false, false>);
    }
    hipLaunchKernelGGL(
        (block_norm_sum_kernel<T>),
        dim3((s.D + 31) / 32, (unsigned)(2 + (pg ? groups : 0))), dim3(1024),
        0, stream.stream(), p1, p2, pg, (const T*)w1.data_ptr(),
        (T*)dw1.data_ptr(), (T*)dw2.data_ptr(), (T*)dg.data_ptr(), grid,
        slices, s.D);
  }))
  HIP_CHECK_LAST();
  return {dh, dx, dw1, dw2, dg};
}
