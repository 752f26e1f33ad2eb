// Rotary positions on one or several axes, for packed tokens.
//
// Frequency j of R/2 turns the pair (x[j], x[j + R/2]) of every head by the
// angle of table row pos[a(j)][token]: its axis a(j) is the section that j
// falls into (time, height, width; one section is the ordinary rotary).
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin     (backward: sin -> -sin)
// Values from R on pass through.
//
// Bound by memory: every value of q and k is read and written once.  A
// thread takes one run of 8 frequencies of one token and turns it in
// several heads of q and k, so that a table row is fetched once for all of
// those heads; 16-byte loads and stores, of any alignment.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_AXES = 4;
constexpr int W = 8;               // frequencies of one thread

struct RopeArgs {
  const void *q, *k;
  void *qo, *ko;                   // contiguous [T, heads, D]
  const void* pos;                 // [axes, T], int32 or int64
  const float *cosb, *sinb;        // [P, R/2]
  long q_t, q_h, k_t, k_h;         // strides of q and k
  long pos_a;                      // stride of an axis of pos
  long T, P;
  int H, HK, D, half, axes, wide_pos;
  int ends[MAX_AXES];              // first frequency behind each section
  float sign;
};

template <class T> __device__ __forceinline__ float up(T v) { return (float)v; }
template <> __device__ __forceinline__ float up(short v) {
  return bf16_to_f32(v);
}
template <class T> __device__ __forceinline__ T down(float f) { return (T)f; }
template <> __device__ __forceinline__ short down(float f) {
  return __builtin_bit_cast(short, (__bf16)f);
}

// 8 values at any alignment of their own type
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Run {
  T v[W];
};

template <class T>
__device__ __forceinline__ void load(const T* p, int n, T (&v)[W]) {
  if (n == W) {
    const Run<T> r = *reinterpret_cast<const Run<T>*>(p);
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = r.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = j < n ? p[j] : (T)0;
  }
}

template <class T>
__device__ __forceinline__ void store(T* p, int n, const T (&v)[W]) {
  if (n == W) {
    Run<T> r;
#pragma unroll
    for (int j = 0; j < W; ++j) r.v[j] = v[j];
    *reinterpret_cast<Run<T>*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j < n) p[j] = v[j];
  }
}

// Work item: (token, part of the heads, run of frequencies or of the values
// that pass through), runs fastest so that neighbouring threads touch
// neighbouring memory.
template <class T>
__global__ __launch_bounds__(NT) void rope_axes_kernel(const RopeArgs a,
                                                       int parts) {
  const int turn_runs = (a.half + W - 1) / W;
  const int pass = a.D - 2 * a.half;
  const int runs = turn_runs + (pass + W - 1) / W;
  const long total = a.T * parts * runs;
  const int heads = a.H + a.HK;
  for (long i = (long)blockIdx.x * NT + threadIdx.x; i < total;
       i += (long)gridDim.x * NT) {
    const int r = (int)(i % runs);
    const int part = (int)(i / runs % parts);
    const long t = i / runs / parts;
    const int h0 = heads * part / parts, h1 = heads * (part + 1) / parts;
    auto from = [&](int h) {
      return h < a.H ? (const T*)a.q + t * a.q_t + h * a.q_h
                     : (const T*)a.k + t * a.k_t + (h - a.H) * a.k_h;
    };
    auto to = [&](int h) {
      return h < a.H ? (T*)a.qo + (t * a.H + h) * a.D
                     : (T*)a.ko + (t * a.HK + h - a.H) * a.D;
    };
    if (r >= turn_runs) {
      const int at = 2 * a.half + (r - turn_runs) * W;
      const int n = min(W, a.D - at);
      for (int h = h0; h < h1; ++h) {
        T v[W];
        load(from(h) + at, n, v);
        store(to(h) + at, n, v);
      }
      continue;
    }
    const int f0 = r * W, n = min(W, a.half - f0);
    float c[W], s[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      c[j] = s[j] = 0.f;
      if (j >= n) continue;
      int axis = 0;
#pragma unroll
      for (int x = 0; x + 1 < MAX_AXES; ++x) axis += f0 + j >= a.ends[x];
      const long o = axis * a.pos_a + t;
      const long p = a.wide_pos ? ((const long*)a.pos)[o]
                                : (long)((const int*)a.pos)[o];
      // a position outside the table has no angle
      const bool ok = p >= 0 && p < a.P;
      const long e = ok ? p * a.half + f0 + j : 0;
      c[j] = ok ? a.cosb[e] : __builtin_nanf("");
      s[j] = ok ? a.sinb[e] * a.sign : __builtin_nanf("");
    }
    for (int h = h0; h < h1; ++h) {
      const T* x = from(h) + f0;
      T* y = to(h) + f0;
      T x1[W], x2[W];
      load(x, n, x1);
      load(x + a.half, n, x2);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float u = up(x1[j]), v = up(x2[j]);
        x1[j] = down<T>(u * c[j] - v * s[j]);
        x2[j] = down<T>(v * c[j] + u * s[j]);
      }
      store(y, n, x1);
      store(y + a.half, n, x2);
    }
  }
}

}  // namespace

// q [T,H,D], k [T,HK,D] (any strides with a dense last dimension), turned
// into new contiguous tensors.
std::vector<torch::Tensor> rope_axes(torch::Tensor q, torch::Tensor k,
                                     torch::Tensor pos, torch::Tensor cosb,
                                     torch::Tensor sinb,
                                     std::vector<int64_t> sections,
                                     bool backward) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3,
              "rope_axes: q and k must be [tokens, heads, dim] on the GPU");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "rope_axes: q and k must have the same tokens and dim");
  const auto st = q.scalar_type();
  TORCH_CHECK((st == torch::kBFloat16 || st == torch::kHalf ||
               st == torch::kFloat32) && k.scalar_type() == st,
              "rope_axes: q and k must both be bf16, fp16 or fp32");
  TORCH_CHECK(q.stride(2) == 1 && k.stride(2) == 1,
              "rope_axes: the last dimension must be dense");
  TORCH_CHECK(cosb.dim() == 2 && cosb.sizes() == sinb.sizes() &&
              cosb.is_contiguous() && sinb.is_contiguous() &&
              cosb.scalar_type() == torch::kFloat32 &&
              sinb.scalar_type() == torch::kFloat32,
              "rope_axes: cos and sin must be contiguous fp32 [places, R/2]");
  TORCH_CHECK(pos.dim() == 2 && pos.size(1) == q.size(0) &&
              pos.is_contiguous() && (pos.scalar_type() == torch::kLong ||
                                      pos.scalar_type() == torch::kInt),
              "rope_axes: positions must be int32 or int64 [axes, tokens]");
  for (const auto& x : {k, pos, cosb, sinb})
    TORCH_CHECK(x.device() == q.device(),
                "rope_axes: all tensors must be on one device");
  RopeArgs a;
  a.axes = (int)sections.size();
  TORCH_CHECK(a.axes >= 1 && a.axes <= MAX_AXES && pos.size(0) == a.axes,
              "rope_axes: 1 to ", MAX_AXES, " sections, a row of positions each");
  a.half = (int)cosb.size(1);
  a.D = (int)q.size(2);
  long sum = 0;
  for (int i = 0; i < MAX_AXES; ++i) {
    TORCH_CHECK(i >= a.axes || sections[i] > 0,
                "rope_axes: sections must be positive");
    sum += i < a.axes ? sections[i] : 0;
    a.ends[i] = i < a.axes ? (int)sum : 1 << 30;
  }
  TORCH_CHECK(sum == a.half && 2 * a.half <= a.D,
              "rope_axes: sections must add up to the tables' width, at most "
              "half of dim");
  const c10::cuda::CUDAGuard guard(q.device());
  auto qo = torch::empty(q.sizes(), q.options());
  auto ko = torch::empty(k.sizes(), k.options());
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.qo = qo.data_ptr();
  a.ko = ko.data_ptr();
  a.pos = pos.data_ptr();
  a.cosb = cosb.data_ptr<float>();
  a.sinb = sinb.data_ptr<float>();
  a.q_t = q.stride(0);
  a.q_h = q.stride(1);
  a.k_t = k.stride(0);
  a.k_h = k.stride(1);
  a.T = q.size(0);
  a.P = cosb.size(0);
  a.pos_a = a.T;
  a.H = (int)q.size(1);
  a.HK = (int)k.size(1);
  a.wide_pos = pos.scalar_type() == torch::kLong;
  a.sign = backward ? -1.f : 1.f;
  const int heads = a.H + a.HK;
  const int runs = (a.half + W - 1) / W + (a.D - 2 * a.half + W - 1) / W;
  if (a.T == 0 || heads == 0) return {qo, ko};
  const int parts = std::max(1, (heads + 7) / 8);
  const long items = a.T * parts * runs;
  const int grid = (int)std::min<long>((items + NT - 1) / NT, 8192);
  auto stream = c10::cuda::getCurrentCUDAStream();
  if (st == torch::kBFloat16)
    hipLaunchKernelGGL((rope_axes_kernel<short>), dim3(grid), dim3(NT), 0,
                       stream.stream(), a, parts);
  else if (st == torch::kHalf)
    hipLaunchKernelGGL((rope_axes_kernel<_Float16>), dim3(grid), dim3(NT), 0,
                       stream.stream(), a, parts);
  else
    hipLaunchKernelGGL((rope_axes_kernel<float>), dim3(grid), dim3(NT), 0,
                       stream.stream(), a, parts);
  HIP_CHECK_LAST();
  return {qo, ko};
}
