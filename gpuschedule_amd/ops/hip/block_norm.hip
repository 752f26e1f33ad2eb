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
// for each block, which a second kernel adds in a fixed order.
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
  return f32_to_bf16(f);
}

template <class T> constexpr int WIDE = 16 / sizeof(T);

// 16 bytes at any alignment of their own type: rows of an odd width begin
// anywhere, and global loads need no alignment beyond that
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Run {
  T v[WIDE<T>];
};

// The values of one row that a thread holds: E values as runs of 16 bytes,
// ROWT threads side by side.
template <class T, int ROWT, int E> struct Row {
  static constexpr int V = WIDE<T>, C = E / V;
  static __device__ __forceinline__ int at(int t, int c) {
    return (c * ROWT + t) * V;
  }
  static __device__ __forceinline__ void load(const T* p, int D, int t,
                                              float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = at(t, c);
      if (i + V <= D) {
        const Run<T> r = *reinterpret_cast<const Run<T>*>(p + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[c * V + j] = up(r.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[c * V + j] = i + j < D ? up(p[i + j]) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, int D, int t,
                                               const float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = at(t, c);
      if (i + V <= D) {
        Run<T> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = down<T>(v[c * V + j]);
        *reinterpret_cast<Run<T>*>(p + i) = r;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (i + j < D) p[i + j] = down<T>(v[c * V + j]);
      }
    }
  }
  static __device__ __forceinline__ void store32(float* p, int D, int t,
                                                 const float (&v)[E]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at(t, c) + j < D) p[at(t, c) + j] = v[c * V + j];
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

template <int ROWT> constexpr int BLOCK = ROWT < 256 ? 256 : ROWT;

// Row i uses row i / group of the gate (no gate: 1).
template <class T, int ROWT, int E>
__global__ __launch_bounds__(BLOCK<ROWT>) void block_norm_fwd_kernel(
    const T* __restrict__ h, const T* __restrict__ x,
    const T* __restrict__ w1, const T* __restrict__ w2,
    const T* __restrict__ gate, T* __restrict__ n_out, T* __restrict__ s_out,
    float* __restrict__ r1_out, float* __restrict__ r2_out, long rows,
    long group, int D, float alpha, float eps) {
  using R = Row<T, ROWT, E>;
  __shared__ float scratch[2][16];
  constexpr int RPB = BLOCK<ROWT> / ROWT;
  const int t = threadIdx.x % ROWT;
  int turn = 0;
  float wa[E], wb[E];
  R::load(w1, D, t, wa);
  R::load(w2, D, t, wb);
  for (long row = (long)blockIdx.x * RPB + threadIdx.x / ROWT; row < rows;
       row += (long)gridDim.x * RPB) {
    float a[E], b[E], g[E];
    R::load(h + row * D, D, t, a);
    R::load(x + row * D, D, t, b);
    if (gate) R::load(gate + row / group * D, D, t, g);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) q += a[i] * a[i];
    const float r1 = rsqrtf(row_sum<ROWT>(q, scratch, turn) / D + eps);
    q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = a[i] * r1 * wa[i];
      b[i] = alpha * b[i] + (gate ? g[i] * z : z);
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

// A worker (the ROWT threads of a row) takes `per` rows in turn.  Where
// `whole`, those are whole groups and each dg row is finished here;
// otherwise they lie in one group, and the worker leaves sum(e hh) behind.
template <class T, int ROWT, int E>
__global__ __launch_bounds__(BLOCK<ROWT>) void block_norm_bwd_kernel(
    const T* __restrict__ dn, const T* __restrict__ ds,
    const T* __restrict__ h, const T* __restrict__ x,
    const T* __restrict__ w1, const T* __restrict__ w2,
    const T* __restrict__ gate, const float* __restrict__ r1s,
    const float* __restrict__ r2s, T* __restrict__ dh, T* __restrict__ dx,
    T* __restrict__ dg, float* __restrict__ part1, float* __restrict__ part2,
    float* __restrict__ partg, long rows, long group, long per, long slices,
    int whole, int D, float alpha) {
  using R = Row<T, ROWT, E>;
  __shared__ float scratch[2][16];
  constexpr int RPB = BLOCK<ROWT> / ROWT;
  const int t = threadIdx.x % ROWT;
  int turn = 0;
  const long worker = (long)blockIdx.x * RPB + threadIdx.x / ROWT;
  long lo, hi;
  if (whole) {
    lo = worker * per;
    hi = min(lo + per, rows);
  } else {                         // `slices` workers share a group
    const long k = worker / slices;
    lo = k * group + worker % slices * per;
    hi = min(lo + per, (k + 1) * group);
    if (k * group >= rows) hi = lo;
  }
  float acc1[E], acc2[E], accg[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc1[i] = acc2[i] = accg[i] = 0.f;
  for (long row = lo; row < hi; ++row) {
    float a[E], b[E], d[E], e[E];
    R::load(h + row * D, D, t, a);
    R::load(x + row * D, D, t, b);
    R::load(dn + row * D, D, t, d);
    R::load(ds + row * D, D, t, e);
    float wa[E], wb[E], g[E];
    R::load(w1, D, t, wa);
    R::load(w2, D, t, wb);
    if (gate) R::load(gate + row / group * D, D, t, g);
    const float r1 = r1s[row], r2 = r2s[row];
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      a[i] *= r1;                  // hh
      const float z = a[i] * wa[i];
      b[i] = (alpha * b[i] + (gate ? g[i] * z : z)) * r2;  // sh
      acc2[i] += d[i] * b[i];
      d[i] *= wb[i];
      q += d[i] * b[i];
    }
    q = row_sum<ROWT>(q, scratch, turn) / D;
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      e[i] += r2 * (d[i] - b[i] * q);
      b[i] = alpha * e[i];
      accg[i] += e[i] * a[i];
      d[i] = (gate ? g[i] * e[i] : e[i]) * wa[i];  // u
      p += d[i] * a[i];
    }
    R::store(dx + row * D, D, t, b);
    p = row_sum<ROWT>(p, scratch, turn) / D;
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] = r1 * (d[i] - a[i] * p);
    R::store(dh + row * D, D, t, d);
    if (row + 1 == hi || (whole && (row + 1) % group == 0)) {
      if (gate && whole) {
#pragma unroll
        for (int i = 0; i < E; ++i) d[i] = wa[i] * accg[i];
        R::store(dg + row / group * D, D, t, d);
      } else if (gate) {
        R::store32(partg + worker * D, D, t, accg);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) {
        acc1[i] += gate ? g[i] * accg[i] : accg[i];
        accg[i] = 0.f;
      }
    }
  }
  if (lo < hi || !whole) {
    R::store32(part1 + worker * D, D, t, acc1);
    R::store32(part2 + worker * D, D, t, acc2);
    if (gate && !whole && lo >= hi) R::store32(partg + worker * D, D, t, accg);
  }
}

// blockIdx.y 0: dw1, 1: dw2, 2 + k: dg of group k, times w1.
template <class T>
__global__ __launch_bounds__(1024) void block_norm_sum_kernel(
    const float* __restrict__ part1, const float* __restrict__ part2,
    const float* __restrict__ partg, const T* __restrict__ w1,
    T* __restrict__ dw1, T* __restrict__ dw2, T* __restrict__ dg, long parts,
    long slices, int D) {
  __shared__ float sh[16][64];
  const int cl = threadIdx.x & 63, pl = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + cl;
  const long k = (long)blockIdx.y - 2;
  const float* p = k < 0 ? (blockIdx.y ? part2 : part1) : partg + k * slices * D;
  const long n = k < 0 ? parts : slices;
  float s = 0.f;
  if (i < D)
    for (long r = pl; r < n; r += 16) s += p[r * D + i];
  sh[pl][cl] = s;
  __syncthreads();
  if (pl != 0 || i >= D) return;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) s += sh[j][cl];
  if (k >= 0) dg[k * D + i] = down<T>(s * up(w1[i]));
  else (blockIdx.y ? dw2 : dw1)[i] = down<T>(s);
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

// Threads of a row: the fewest that hold it at 16 values each.
#define BY_WIDTH(T, D, ...)                                             \
  if ((D) <= 64 * 8) { constexpr int ROWT = 64, E = 8; __VA_ARGS__; }   \
  else if ((D) <= 64 * 16) { constexpr int ROWT = 64, E = 16; __VA_ARGS__; } \
  else if ((D) <= 256 * 8) { constexpr int ROWT = 256, E = 8; __VA_ARGS__; } \
  else if ((D) <= 256 * 16) { constexpr int ROWT = 256, E = 16; __VA_ARGS__; } \
  else if ((D) <= 512 * 16) { constexpr int ROWT = 512, E = 16; __VA_ARGS__; } \
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
    const int grid = (int)std::min<long>((s.rows + RPB - 1) / RPB, 8192);
    hipLaunchKernelGGL((block_norm_fwd_kernel<T, ROWT, E>), dim3(grid),
                       dim3(BLOCK<ROWT>), 0, stream.stream(),
                       (const T*)h.data_ptr(), (const T*)x.data_ptr(),
                       (const T*)w1.data_ptr(), (const T*)w2.data_ptr(),
                       gate ? (const T*)gate->data_ptr() : nullptr,
                       (T*)n.data_ptr(), (T*)sum.data_ptr(),
                       train ? r1.data_ptr<float>() : nullptr,
                       train ? r2.data_ptr<float>() : nullptr, s.rows,
                       s.group, s.D, (float)alpha, (float)eps);
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
  // About 1024 rows of 256 threads at work fill the card, each adding one
  // partial row: a group of rows is cut into as many slices as that allows,
  // and a worker takes several whole groups where there are more.
  BY_TYPE(h.scalar_type(), BY_WIDTH(T, s.D, {
    constexpr int RPB = BLOCK<ROWT> / ROWT;
    const long want = std::min<long>(s.rows, 1024L * RPB * 256 / BLOCK<ROWT>);
    const int whole = groups >= want;
    long per = 0;
    long slices = 1;
    long workers = 0;
    if (whole) {
      per = (groups + want - 1) / want * s.group;
      workers = (s.rows + per - 1) / per;
    } else {
      slices = std::max<long>(1, want / groups);
      per = (s.group + slices - 1) / slices;
      slices = (s.group + per - 1) / per;
      workers = groups * slices;
    }
    const long grid = (workers + RPB - 1) / RPB;
    auto fopt = h.options().dtype(torch::kFloat32);
    auto part = torch::empty({gate && !whole ? 3 : 2, grid * RPB, s.D}, fopt);
    float* p1 = part.data_ptr<float>();
    float* p2 = p1 + grid * RPB * s.D;
    float* pg = gate && !whole ? p2 + grid * RPB * s.D : nullptr;
    hipLaunchKernelGGL(
        (block_norm_bwd_kernel<T, ROWT, E>), dim3((unsigned)grid),
        dim3(BLOCK<ROWT>), 0, stream.stream(), (const T*)dn.data_ptr(),
        (const T*)ds.data_ptr(), (const T*)h.data_ptr(),
        (const T*)x.data_ptr(), (const T*)w1.data_ptr(),
        (const T*)w2.data_ptr(),
        gate ? (const T*)gate->data_ptr() : nullptr, r1.data_ptr<float>(),
        r2.data_ptr<float>(), (T*)dh.data_ptr(), (T*)dx.data_ptr(),
        (T*)dg.data_ptr(), p1, p2, pg, s.rows, s.group, per, slices, whole,
        s.D, (float)alpha);
    hipLaunchKernelGGL(
        (block_norm_sum_kernel<T>),
        dim3((s.D + 63) / 64, (unsigned)(2 + (pg ? groups : 0))), dim3(1024),
        0, stream.stream(), p1, p2, pg, (const T*)w1.data_ptr(),
        (T*)dw1.data_ptr(), (T*)dw2.data_ptr(), (T*)dg.data_ptr(), workers,
        slices, s.D);
  }))
  HIP_CHECK_LAST();
  return {dh, dx, dw1, dw2, dg};
}
