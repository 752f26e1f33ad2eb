// Global gradient norm over many tensors, and clipping by it.
//
//   N = sqrt(sum over all tensors of g^2),  g <- g * min(1, max / (N + 1e-6))
//
// Two launches for up to MAX_T tensors, whatever their sizes and types:
// the first sums squares, the second joins the partial sums and scales.
// Pointers travel in the kernel arguments, so a call copies nothing to the
// device and a captured graph replays on the same gradients.
//
// Squares are summed in 64 bits: the square of any fp32 value is in range
// there, so N is right wherever N itself is, for gradients of 1e-30 as for
// those of 1e30.  Every block writes its own partial and every joiner adds
// them in the same order: the result does not change from run to run.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_T = 192;         // tensors of one launch: 3.3 KB of arguments
constexpr long CHUNK = 8192;       // values of one piece of work
constexpr int MAX_BLOCKS = 2048;   // 8 blocks of 4 waves on each CU
enum { BF16 = 0, F16 = 1, F32 = 2 };

struct GradTable {
  void* ptr[MAX_T];
  unsigned numel[MAX_T];
  unsigned first[MAX_T + 1];       // first chunk of each tensor, and the end
  unsigned char type[MAX_T];
  int count;
};

template <int TYPE> struct Elem;
template <> struct Elem<BF16> {
  using T = short;
  static __device__ float up(T v) { return bf16_to_f32(v); }
  static __device__ T down(float f) {
    return __builtin_bit_cast(short, (__bf16)f);
  }
};
template <> struct Elem<F16> {
  using T = _Float16;
  static __device__ float up(T v) { return (float)v; }
  static __device__ T down(float f) { return (_Float16)f; }
};
template <> struct Elem<F32> {
  using T = float;
  static __device__ float up(T v) { return v; }
  static __device__ T down(float f) { return f; }
};

// Calls one(value) for the values before the first and behind the last
// 16-byte line of p[0..n), and line(16 bytes) for the lines between.
template <int TYPE, class One, class Line>
__device__ __forceinline__ void each(typename Elem<TYPE>::T* p, unsigned n,
                                     One one, Line line) {
  using T = typename Elem<TYPE>::T;
  constexpr unsigned V = 16 / sizeof(T);
  unsigned head = (unsigned)((16 - ((size_t)p & 15)) & 15) / sizeof(T);
  head = min(head, n);
  const unsigned lines = (n - head) / V, tail = head + lines * V;
  if (threadIdx.x < head) one(p[threadIdx.x]);
  if (threadIdx.x < n - tail) one(p[tail + threadIdx.x]);
  typedef __attribute__((ext_vector_type(V))) T VT;
  VT* q = reinterpret_cast<VT*>(p + head);
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < lines; i += NT) line(q[i]);
}

template <int TYPE>
__device__ __forceinline__ double squares(void* ptr, unsigned n) {
  using E = Elem<TYPE>;
  double s = 0.0;
  auto one = [&](typename E::T& v) {
    const double f = E::up(v);
    s += f * f;
  };
  each<TYPE>((typename E::T*)ptr, n, one, [&](auto& v) {
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(typename E::T)); ++j) {
      const double f = E::up(v[j]);
      s += f * f;
    }
  });
  return s;
}

template <int TYPE>
__device__ __forceinline__ void scale(void* ptr, unsigned n, float c) {
  using E = Elem<TYPE>;
  each<TYPE>((typename E::T*)ptr, n,
             [&](typename E::T& v) { v = E::down(E::up(v) * c); },
             [&](auto& v) {
               auto w = v;
#pragma unroll
               for (int j = 0; j < (int)(16 / sizeof(typename E::T)); ++j)
                 w[j] = E::down(E::up(w[j]) * c);
               v = w;
             });
}

// The sum of one double of each thread, in every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[NT / WAVE];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < NT / WAVE; ++w) v += part[w];
  __syncthreads();
  return v;
}

// A block takes a run of neighbouring chunks: one search for the tensor of
// its first chunk, then it walks on.
__device__ __forceinline__ int tensor_of(const GradTable& t, unsigned chunk) {
  int lo = 0, hi = t.count - 1;  // the last tensor that begins at or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(NT) void grad_squares_kernel(
    const GradTable t, double* __restrict__ part) {
  const unsigned chunks = t.first[t.count];
  const unsigned c0 = (unsigned)((unsigned long)chunks * blockIdx.x / gridDim.x);
  const unsigned c1 =
      (unsigned)((unsigned long)chunks * (blockIdx.x + 1) / gridDim.x);
  int k = tensor_of(t, c0);
  double s = 0.0;
  for (unsigned c = c0; c < c1; ++c) {
    while (t.first[k + 1] <= c) ++k;
    const size_t off = (size_t)(c - t.first[k]) * CHUNK;
    const unsigned n = (unsigned)min((size_t)CHUNK, t.numel[k] - off);
    if (t.type[k] == BF16) s += squares<BF16>((short*)t.ptr[k] + off, n);
    else if (t.type[k] == F16) s += squares<F16>((_Float16*)t.ptr[k] + off, n);
    else s += squares<F32>((float*)t.ptr[k] + off, n);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double joined_norm(const double* __restrict__ part,
                                              int parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += NT) s += part[i];
  return sqrt(block_sum(s));
}

__global__ __launch_bounds__(NT) void grad_norm_kernel(
    const double* __restrict__ part, int parts, float* __restrict__ norm) {
  const double n = joined_norm(part, parts);
  if (threadIdx.x == 0) norm[0] = (float)n;
}

__global__ __launch_bounds__(NT) void grad_clip_kernel(
    const GradTable t, const double* __restrict__ part, int parts,
    double max_norm, float* __restrict__ norm) {
  const double n = joined_norm(part, parts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
  const double ratio = max_norm / (n + 1e-6);
  if (ratio >= 1.0) return;        // nothing to clip (NaN goes on, and spreads)
  const float c = (float)ratio;
  const unsigned chunks = t.first[t.count];
  const unsigned c0 = (unsigned)((unsigned long)chunks * blockIdx.x / gridDim.x);
  const unsigned c1 =
      (unsigned)((unsigned long)chunks * (blockIdx.x + 1) / gridDim.x);
  int k = tensor_of(t, c0);
  for (unsigned i = c0; i < c1; ++i) {
    while (t.first[k + 1] <= i) ++k;
    const size_t off = (size_t)(i - t.first[k]) * CHUNK;
    const unsigned m = (unsigned)min((size_t)CHUNK, t.numel[k] - off);
    if (t.type[k] == BF16) scale<BF16>((short*)t.ptr[k] + off, m, c);
    else if (t.type[k] == F16) scale<F16>((_Float16*)t.ptr[k] + off, m, c);
    else scale<F32>((float*)t.ptr[k] + off, m, c);
  }
}

struct Grad {
  char *begin, *end;
  at::TensorImpl *param, *grad;
  int type;
};

// The gradients of `params`, each once, in the order of their addresses.
std::vector<Grad> grads_of(const std::vector<torch::Tensor>& params) {
  std::vector<Grad> grads;
  grads.reserve(params.size());
  c10::optional<c10::Device> device;
  for (const auto& p : params) {
    const auto& g = p.grad();
    if (!g.defined()) continue;
    if (!device) device = g.device();
    TORCH_CHECK(g.is_cuda() && g.device() == *device,
                "grad_norm: all gradients must be on one GPU");
    TORCH_CHECK(g.layout() == torch::kStrided && g.is_non_overlapping_and_dense(),
                "grad_norm: gradients must be dense in memory");
    const auto st = g.scalar_type();
    TORCH_CHECK(st == torch::kBFloat16 || st == torch::kHalf ||
                    st == torch::kFloat32,
                "grad_norm: gradients must be bf16, fp16 or fp32, got ", st);
    TORCH_CHECK(!g._fw_grad(0).defined(),
                "grad_norm: gradients with a forward-mode tangent are not "
                "supported");
    if (g.numel() == 0) continue;
    char* at = (char*)g.data_ptr();
    grads.push_back({at, at + g.nbytes(), p.unsafeGetTensorImpl(),
                     g.unsafeGetTensorImpl(),
                     st == torch::kBFloat16 ? BF16
                                            : st == torch::kHalf ? F16 : F32});
  }
  std::sort(grads.begin(), grads.end(), [](const Grad& a, const Grad& b) {
    return a.begin < b.begin;
  });
  // a tied weight counts once
  grads.erase(std::unique(grads.begin(), grads.end(),
                          [](const Grad& a, const Grad& b) {
                            return a.param == b.param;
                          }),
              grads.end());
  // two blocks would scale shared memory at once
  for (size_t i = 1; i < grads.size(); ++i)
    TORCH_CHECK(grads[i].begin >= grads[i - 1].end,
                "grad_norm: two gradients share memory");
  return grads;
}

std::vector<GradTable> tables_of(const std::vector<Grad>& grads) {
  constexpr long PIECE = 1L << 30;  // a longer tensor takes several entries
  std::vector<GradTable> tables;
  for (const auto& g : grads) {
    const long size = g.type == F32 ? 4 : 2, n = (g.end - g.begin) / size;
    for (long off = 0; off < n; off += PIECE) {
      if (tables.empty() || tables.back().count == MAX_T) {
        tables.emplace_back();
        tables.back().count = 0;
        tables.back().first[0] = 0;
      }
      auto& t = tables.back();
      const long m = std::min(PIECE, n - off);
      const int i = t.count++;
      t.ptr[i] = g.begin + off * size;
      t.numel[i] = (unsigned)m;
      t.type[i] = g.type;
      t.first[i + 1] = t.first[i] + (unsigned)((m + CHUNK - 1) / CHUNK);
    }
  }
  return tables;
}

}  // namespace

// The norm of the gradients of `params`, as fp32 [] (those without one are
// left out).  max_norm >= 0: they are scaled in place so that their norm is
// at most that.  max_norm < 0: norm only.
torch::Tensor grad_norm_clip(std::vector<torch::Tensor> params,
                             double max_norm) {
  c10::optional<torch::Tensor> any;
  for (const auto& p : params)
    if (p.grad().defined()) any = p.grad();
  TORCH_CHECK(any, "grad_norm: no gradients");
  const auto grads = grads_of(params);
  const auto tables = tables_of(grads);
  const c10::cuda::CUDAGuard guard(any->device());
  auto stream = c10::cuda::getCurrentCUDAStream();
  const auto opt = torch::TensorOptions().device(any->device());
  auto norm = torch::empty({}, opt.dtype(torch::kFloat32));
  std::vector<int> grid;
  int parts = 0;
  for (const auto& t : tables) {
    grid.push_back((int)std::min<unsigned>(t.first[t.count], MAX_BLOCKS));
    parts += grid.back();
  }
  auto part = torch::empty({std::max(parts, 1)}, opt.dtype(torch::kFloat64));
  double* pp = part.data_ptr<double>();
  int at = 0;
  for (size_t i = 0; i < tables.size(); ++i) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(grid[i]), dim3(NT), 0,
                       stream.stream(), tables[i], pp + at);
    at += grid[i];
  }
  if (max_norm < 0 || tables.empty())
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(NT), 0,
                       stream.stream(), pp, parts, norm.data_ptr<float>());
  else
    for (size_t i = 0; i < tables.size(); ++i)
      hipLaunchKernelGGL(grad_clip_kernel, dim3(grid[i]), dim3(NT), 0,
                         stream.stream(), tables[i], pp, parts, max_norm,
                         i == 0 ? norm.data_ptr<float>() : nullptr);
  if (max_norm >= 0)
    for (const auto& g : grads)
      if (!g.grad->is_inference()) g.grad->bump_version();
  HIP_CHECK_LAST();
  return norm;
}
