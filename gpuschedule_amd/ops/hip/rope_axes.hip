// Rotary positions on one or several axes, for packed tokens.
//
// Frequency j of R/2 turns the pair (x[j], x[j + R/2]) of every head by the
// angle of table row pos[a(j)][token]: its axis a(j) is the section that j
// falls into (time, height, width; one section is the ordinary rotary).
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin     (backward: sin -> -sin)
// Values from R on pass through.
//
// Bound by memory: every value of q and k is read and written once.  A
// thread takes one run of 8 frequencies of one token and turns it in four
// heads, so that a table row is fetched once for those; loads and stores of
// 8 values at any alignment.  16384 tokens, 32 and 8 heads of 128 bf16 (335
// MB): 69 us, 4.8 TB/s, as a copy.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_AXES = 4;
constexpr int W = 8;               // frequencies of one thread
constexpr int HPT = 4;             // heads of one thread: a table row is
// fetched once for them (one head each: 10.8 us for 1024 tokens of 32 and 8
// heads of 128 and 34 for 8192; four: 8.6 and 32)

struct RopeArgs {
  const void *q, *k;
  void *qo, *ko;                   // contiguous [T, heads, D]
  const void* pos;                 // [axes, T], int32 or int64
  const float *cosb, *sinb;        // [P, R/2]
  long q_t, q_h, k_t, k_h;         // strides of q and k
  long T, P;
  long rows;                       // tokens of one value of blockIdx.y
  int H, HK, D, half, axes, wide_pos;
  int ends[MAX_AXES];              // first frequency behind each section
  float sign;
};

template <class T> __device__ __forceinline__ T down(float f) { return (T)f; }
template <> __device__ __forceinline__ short down(float f) {
  return __builtin_bit_cast(short, (__bf16)f);
}

template <class T> __device__ __forceinline__ unsigned bits_of(T v) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(unsigned, v);
  else return __builtin_bit_cast(unsigned short, v);
}

// 8 values at any alignment of their own type, 16-bit ones two to a register
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Run {
  static constexpr int PER = 4 / sizeof(T), N = W / PER;
  unsigned w[N];

  __device__ __forceinline__ float get(int j) const {
    const unsigned u = w[j / PER];
    if constexpr (std::is_same_v<T, float>) return __builtin_bit_cast(float, u);
    else if constexpr (std::is_same_v<T, short>)
      return __builtin_bit_cast(float, j & 1 ? u & 0xffff0000u : u << 16);
    else
      return (float)__builtin_bit_cast(
          _Float16, (unsigned short)(j & 1 ? u >> 16 : u));
  }
  __device__ __forceinline__ void set(const float (&f)[W]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = bits_of(down<T>(f[i * PER]));
      if constexpr (PER == 2) w[i] |= bits_of(down<T>(f[i * 2 + 1])) << 16;
    }
  }
};

template <class T> __device__ __forceinline__ Run<T> load(const T* p, int n) {
  if (n == W) return *reinterpret_cast<const Run<T>*>(p);
  Run<T> r = {};
  constexpr int PER = Run<T>::PER;
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < n) r.w[j / PER] |= bits_of(p[j]) << (j % PER * 16);
  return r;
}

template <class T>
__device__ __forceinline__ void store(T* p, int n, const Run<T>& r) {
  if (n == W) {
    *reinterpret_cast<Run<T>*>(p) = r;
  } else {
    constexpr int PER = Run<T>::PER;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const unsigned u = r.w[j / PER] >> (j % PER * 16);
      if constexpr (PER == 1) {
        if (j < n) p[j] = __builtin_bit_cast(T, u);
      } else {
        if (j < n) p[j] = __builtin_bit_cast(T, (unsigned short)u);
      }
    }
  }
}

// Work item: (token, HPT heads of q or of k, run of frequencies or of the
// values that pass through), runs fastest so that neighbouring threads touch
// neighbouring memory.  All of an item's loads are issued before its first
// store.
template <class T>
__global__ __launch_bounds__(NT) void rope_axes_kernel(const RopeArgs a,
                                                       int runs, int q_parts,
                                                       int parts) {
  const int turn_runs = (a.half + W - 1) / W;
  const unsigned i = blockIdx.x * NT + threadIdx.x;
  const unsigned r = i % runs, rest = i / runs;
  const unsigned part = rest % parts;
  const long t = (long)blockIdx.y * a.rows + rest / parts;
  if (rest / parts >= a.rows || t >= a.T) return;
  const bool is_q = (int)part < q_parts;
  const int heads = is_q ? a.H : a.HK;
  const int h0 = (is_q ? part : part - q_parts) * HPT;
  const long step = is_q ? a.q_h : a.k_h;
  const T* x = is_q ? (const T*)a.q + t * a.q_t : (const T*)a.k + t * a.k_t;
  T* y = is_q ? (T*)a.qo : (T*)a.ko;
  const bool turned = (int)r < turn_runs;
  const int f0 = turned ? r * W : 2 * a.half + (r - turn_runs) * W;
  const int n = min(W, turned ? a.half - f0 : a.D - f0);
  x += h0 * step + f0;
  y += (t * heads + h0) * a.D + f0;
  const int far = turned ? a.half : 0;  // to the pair's other value
  Run<T> u[HPT], v[HPT];
#pragma unroll
  for (int h = 0; h < HPT; ++h)
    if (h0 + h < heads) {
      u[h] = load(x + h * step, n);
      if (turned) v[h] = load(x + h * step + far, n);
    }
  if (turned) {
    auto axis_of = [&](int f) {
      int axis = 0;
#pragma unroll
      for (int e = 0; e + 1 < MAX_AXES; ++e) axis += f >= a.ends[e];
      return axis;
    };
    auto position = [&](int axis) {
      const long o = axis * a.T + t;
      return a.wide_pos ? ((const long*)a.pos)[o]
                        : (long)((const int*)a.pos)[o];
    };
    // a position outside the table has no angle
    float c[W], s[W];
    const int axis = axis_of(f0);
    if (n == W && axis == axis_of(f0 + W - 1)) {
      const long p = position(axis);
      const bool ok = p >= 0 && p < a.P;
      const long e = (ok ? p : 0) * a.half + f0;
      Run<float> cr = {}, sr = {};
      if (ok) {
        cr = load(a.cosb + e, W);
        sr = load(a.sinb + e, W);
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        c[j] = ok ? cr.get(j) : __builtin_nanf("");
        s[j] = sr.get(j) * a.sign;
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        c[j] = s[j] = 0.f;
        if (j >= n) continue;
        const long p = position(axis_of(f0 + j));
        const bool ok = p >= 0 && p < a.P;
        const long e = p * a.half + f0 + j;
        c[j] = ok ? a.cosb[e] : __builtin_nanf("");
        s[j] = ok ? a.sinb[e] * a.sign : 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
      float p[W], q[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        p[j] = u[h].get(j) * c[j] - v[h].get(j) * s[j];
        q[j] = v[h].get(j) * c[j] + u[h].get(j) * s[j];
      }
      u[h].set(p);
      v[h].set(q);
    }
  }
#pragma unroll
  for (int h = 0; h < HPT; ++h)
    if (h0 + h < heads) {
      store(y + (long)h * a.D, n, u[h]);
      if (turned) store(y + (long)h * a.D + far, n, v[h]);
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
  a.H = (int)q.size(1);
  a.HK = (int)k.size(1);
  a.wide_pos = pos.scalar_type() == torch::kLong;
  a.sign = backward ? -1.f : 1.f;
  if (a.T == 0 || a.H + a.HK == 0) return {qo, ko};
  const int runs = (a.half + W - 1) / W + (a.D - 2 * a.half + W - 1) / W;
  auto stream = c10::cuda::getCurrentCUDAStream();
  const int q_parts = (a.H + HPT - 1) / HPT;
  const int parts = q_parts + (a.HK + HPT - 1) / HPT;
  const long per = (long)parts * runs;     // items of a token
  TORCH_CHECK(per < (1L << 30), "rope_axes: too many heads");
  a.rows = std::max<long>(1, std::min<long>(a.T, (1L << 30) / per));
  const dim3 grid((unsigned)((a.rows * per + NT - 1) / NT),
                  (unsigned)((a.T + a.rows - 1) / a.rows));
  TORCH_CHECK(grid.y < 65536, "rope_axes: too many tokens and heads");
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, stream.stream(), a, runs,
                       q_parts, parts);
  };
  if (st == torch::kBFloat16) launch(rope_axes_kernel<short>);
  else if (st == torch::kHalf) launch(rope_axes_kernel<_Float16>);
  else launch(rope_axes_kernel<float>);
  HIP_CHECK_LAST();
  return {qo, ko};
}
