// Muon: momentum, orthogonalised update and weight update of matrices (sm_100a).
//
// For a matrix W with gradient G (K. Jordan's Muon; the momentum form of torch.optim.Muon):
//     M <- mu M + (1 - mu) G,   U = (1 - mu) G + mu M  (look-ahead)  or  U = M
//     O = five Newton-Schulz steps of U / max(|U|_F, eps)                (newton_schulz.cu)
//     W <- W (1 - lr wd) - lr s O
//
// The element-wise kernels here are bound by HBM: per element of bf16 parameters the momentum kernel
// moves 10 bytes (G, M read, M written) and sums U's squares; the load kernel reads G and M again
// (6 bytes; U itself is never stored, which would round it before its norm is known) and writes
// the two fp16 planes of U / |U|; the weight kernel reads O and the master and writes the master and
// the changed sectors of the copy.  Measured on 12288 x 4096 of bf16: momentum 79 us (6.4 TB/s), load 74 us
// (6.8 TB/s).  A launch takes its matrices' descriptors as kernel parameters
// (kSlice of them, of any shapes), so a step uploads no table and can be captured into a graph.
//
// Sums: squares are taken and added in fp64 (gradients of 1e-30 or 1e25 keep their norm), each CTA
// writes its own partial, and every reader adds a matrix's partials in the same order, so results
// do not depend on scheduling.
#include <cmath>

#include "ha_common.cuh"
#include "ha_param.cuh"
#include "newton_schulz.cuh"
#include "umma.cuh"

namespace ha {
namespace {

constexpr int kSlice = 32;               // tensors of one launch: 32 x 120 bytes of kernel parameters
constexpr int64_t kMinChunk = 8192;      // elements of one partial sum at least
constexpr int64_t kMaxPartials = 512;    // partial sums of one matrix at most
constexpr int kLoadChunk = kThreads * 8 * 4;  // padded elements of a CTA of the load and store kernels
constexpr int64_t kApplyChunk = 16384;
// 4-element groups per thread and pass of the weight kernel: 361 us for 193 M bf16 weights (2.3 GB, 6.4 TB/s);
// 4 take 475 us and 8 take 598: fewer CTAs fit an SM.
constexpr int kGroups = 2;
constexpr int64_t kMaxPass = 4096;       // matrices of one pass
// Up to this size one CTA sums, updates and loads a matrix in one launch.  Two launches / one, us of a whole call: one of
// 64 x 96 35.7 / 31.8, 128 x 128 53.4 / 49.6, 128 x 256 60.8 / 59.8, 192 x 256 81.2 / 82.7, 256 x 256 85.0 / 89.1;
// 16 of 128 x 256 62.2 / 61.7, 256 x 256 90.6 / 92.7.
constexpr int64_t kWholeElems = 32768;
constexpr int kWholeThreads = 1024;
constexpr int64_t kSliceBytes = 48 << 20;  // of matrices between the two reads of a slice: they stay in L2
constexpr size_t kHeader = 256 + kMaxPass * 4;  // the workspace's error word, the matrices' counters

// A matrix of a launch and its workspace; matrices of any shapes share launches.
struct Entry {
  ha_tensor t;
  double* partials;
  uint32_t* counter;
  __half *hi, *lo;  // X's planes (weight kernel: hi holds the result)
  uint32_t rows, cols, ld;
  int32_t n_partials;
  int64_t chunk;    // elements of a partial sum
};
struct Slice {
  Entry e[kSlice];
};

struct MuonConst {
  float mu, a_mu;  // mu and 1 - mu
  int nesterov, use_decay, clip;
  float clip_mult;
};

int64_t chunk_for(int64_t numel) {
  const int64_t c = (numel + kMaxPartials - 1) / kMaxPartials;
  return (c + kMinChunk - 1) / kMinChunk * kMinChunk;
}

template <int THREADS = kThreads>
__device__ __forceinline__ double block_sum_all(double x, double* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) smem[warp] = x;
  __syncthreads();
  x = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) x += smem[w];
  return x;  // in every thread
}

// Eight consecutive elements of a DT array (a 16-byte aligned address) as fp32.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::raw* p, float (&x)[8]) {
  if constexpr (DT == HA_F32) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Elem<DT>::widen(uint16_t(v[i] & 0xffffu));
      x[2 * i + 1] = Elem<DT>::widen(uint16_t(v[i] >> 16));
    }
  }
}

__device__ __forceinline__ void add_square(double& acc, float u) {
  const double d = double(u);
  acc = __fma_rn(d, d, acc);
}

// One element of the momentum and of the update direction.
template <int DT>
__device__ __forceinline__ float momentum_elem(const MuonConst& s, float g, float& m) {
  if (s.clip) g = clip_round<DT>(g, s.clip_mult);
  m = __fmaf_rn(s.a_mu, g, __fmul_rn(m, s.mu));
  return s.nesterov ? __fmaf_rn(s.a_mu, g, __fmul_rn(m, s.mu)) : m;
}
// The direction from the momentum already updated.
template <int DT>
__device__ __forceinline__ float direction_elem(const MuonConst& s, float g, float m) {
  if (!s.nesterov) return m;
  if (s.clip) g = clip_round<DT>(g, s.clip_mult);
  return __fmaf_rn(s.a_mu, g, __fmul_rn(m, s.mu));
}

// Square sums of plain matrices, `numel` elements each, one after another.  Grid: (partials, matrices).
template <int DT>
__global__ void __launch_bounds__(kThreads)
    square_sum_kernel(const void* src, int64_t numel, int64_t chunk, double* partials, uint32_t* error) {
  __shared__ double red[kThreads / 32];
  using raw = typename Elem<DT>::raw;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && error != nullptr) *error = 0;
  const raw* x = static_cast<const raw*>(src) + int64_t(blockIdx.y) * numel;
  const int64_t begin = int64_t(blockIdx.x) * chunk, end = min(begin + chunk, numel);
  double acc = 0.0;
  int64_t e = begin + int64_t(threadIdx.x) * 8;
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
    for (; e + 8 <= end; e += kThreads * 8) {
      float v[8];
      load8<DT>(x + e, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) add_square(acc, v[i]);
    }
    for (int64_t k = e; k < min(e + 8, end); ++k) add_square(acc, Elem<DT>::widen(x[k]));
  } else {
    for (int64_t k = begin + threadIdx.x; k < end; k += kThreads) add_square(acc, Elem<DT>::widen(x[k]));
  }
  acc = block_sum_all(acc, red);
  if (threadIdx.x == 0) partials[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = acc;
}

// Momentum update and square sums of the direction.  Grid: (most partials of a matrix, matrices).
template <int DT>
__global__ void __launch_bounds__(kThreads)
    momentum_kernel(const __grid_constant__ Slice s, MuonConst c, uint32_t* error) {
  __shared__ double red[kThreads / 32];
  using raw = typename Elem<DT>::raw;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && error != nullptr) *error = 0;
  const Entry& entry = s.e[blockIdx.y];
  if (int(blockIdx.x) >= entry.n_partials) return;
  const ha_tensor& t = entry.t;
  const raw* grad = reinterpret_cast<const raw*>(t.grad);
  float* mom = reinterpret_cast<float*>(t.exp_avg);
  const int64_t begin = int64_t(blockIdx.x) * entry.chunk, end = min(begin + entry.chunk, t.numel);
  double acc = 0.0;
  auto one = [&](int64_t k) {
    float m = mom[k];
    add_square(acc, momentum_elem<DT>(c, Elem<DT>::widen(grad[k]), m));
    mom[k] = m;
  };
  if (((t.grad | t.exp_avg) & 15) == 0) {
    int64_t e = begin + int64_t(threadIdx.x) * 8;
    for (; e + 8 <= end; e += kThreads * 8) {
      float g[8], m[8];
      load8<DT>(grad + e, g);
      load8<HA_F32>(mom + e, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) add_square(acc, momentum_elem<DT>(c, g[i], m[i]));
      reinterpret_cast<float4*>(mom + e)[0] = make_float4(m[0], m[1], m[2], m[3]);
      reinterpret_cast<float4*>(mom + e)[1] = make_float4(m[4], m[5], m[6], m[7]);
    }
    for (int64_t k = e; k < min(e + 8, end); ++k) one(k);
  } else {
    for (int64_t k = begin + threadIdx.x; k < end; k += kThreads) one(k);
  }
  acc = block_sum_all(acc, red);
  if (threadIdx.x == 0) entry.partials[blockIdx.x] = acc;
}

struct Shape {
  int64_t rows, cols, ld, plane;
};

// A matrix for the load kernel.
struct Target {
  const double* partials;
  uint32_t* counter;
  __half *hi, *lo;
  uint32_t rows, cols, ld;
  int n_partials;
};

// What the load kernel reads: element k of matrix `y` of the launch.
template <int DT>
struct PlainSource {
  const typename Elem<DT>::raw* x;
  int64_t numel, plane;
  Target first;
  struct View {
    const typename Elem<DT>::raw* x;
    __device__ bool aligned() const { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
    __device__ float one(int64_t k) const { return Elem<DT>::widen(x[k]); }
    __device__ void eight(int64_t k, float (&v)[8]) const { load8<DT>(x + k, v); }
    // The first visit of an element (whole_kernel).
    __device__ float first_one(int64_t k) const { return one(k); }
    __device__ void first_eight(int64_t k, float (&v)[8]) const { eight(k, v); }
  };
  __device__ View view(int y) const { return View{x + y * numel}; }
  __device__ Target target(int y) const {
    Target t = first;
    t.partials += int64_t(y) * t.n_partials;
    t.counter += y;
    t.hi += y * plane;
    t.lo += y * plane;
    return t;
  }
};
template <int DT>
struct MuonSource {
  Slice s;
  MuonConst c;
  struct View {
    const typename Elem<DT>::raw* g;
    float* m;
    MuonConst c;
    __device__ bool aligned() const {
      return ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m)) & 15) == 0;
    }
    __device__ float one(int64_t k) const { return direction_elem<DT>(c, Elem<DT>::widen(g[k]), m[k]); }
    __device__ void eight(int64_t k, float (&v)[8]) const {
      float a[8];
      load8<DT>(g + k, a);
      load8<HA_F32>(m + k, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = direction_elem<DT>(c, a[i], v[i]);
    }
    // The first visit updates the momentum.
    __device__ float first_one(int64_t k) const {
      float w = m[k];
      const float u = momentum_elem<DT>(c, Elem<DT>::widen(g[k]), w);
      m[k] = w;
      return u;
    }
    __device__ void first_eight(int64_t k, float (&v)[8]) const {
      float a[8], w[8];
      load8<DT>(g + k, a);
      load8<HA_F32>(m + k, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = momentum_elem<DT>(c, a[i], w[i]);
      reinterpret_cast<float4*>(m + k)[0] = make_float4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<float4*>(m + k)[1] = make_float4(w[4], w[5], w[6], w[7]);
    }
  };
  __device__ View view(int y) const {
    return View{reinterpret_cast<const typename Elem<DT>::raw*>(s.e[y].t.grad),
                reinterpret_cast<float*>(s.e[y].t.exp_avg), c};
  }
  __device__ Target target(int y) const {
    const Entry& e = s.e[y];
    return Target{e.partials, e.counter, e.hi, e.lo, e.rows, e.cols, e.ld, e.n_partials};
  }
};

// Eight padded elements of a matrix, X0 = U / max(|U|_F, eps), into its high and low planes (row padding
// holds zeros).
template <class View>
__device__ __forceinline__ void load_group(const Target& m, const View& v, bool vec, float scale, uint32_t per_row,
                                           int64_t k) {
  const uint32_t r = uint32_t(k) / per_row, c = (uint32_t(k) - r * per_row) * 8;
  const int64_t e = int64_t(r) * m.cols + c;
  float x[8];
  if (vec) {
    v.eight(e, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < m.cols ? v.one(e + i) : 0.0f;
  }
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __fmul_rn(x[2 * i], scale), b = __fmul_rn(x[2 * i + 1], scale);
    const __half2 p = __floats2half2_rn(a, b);
    const float2 f = __half22float2(p);
    const __half2 q = __floats2half2_rn((a - f.x) * kScaleLo, (b - f.y) * kScaleLo);
    h[i] = *reinterpret_cast<const uint32_t*>(&p);
    l[i] = *reinterpret_cast<const uint32_t*>(&q);
  }
  const int64_t at = int64_t(r) * m.ld + c;
  *reinterpret_cast<uint4*>(m.hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(m.lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ float scale_of(double sum, double eps) {
  const double norm = sqrt(sum);
  return float(double(kScaleX) / (norm < eps ? eps : norm));  // a NaN norm stays one
}

// Grid: (most chunks of a padded matrix, matrices); the square sums are there.
template <class Source>
__global__ void __launch_bounds__(kThreads) load_kernel(const __grid_constant__ Source src, double eps) {
  __shared__ double red[kThreads / 32];
  grid_launch_dependents();
  const Target m = src.target(blockIdx.y);
  const uint32_t per_row = m.ld >> 3;
  const int64_t total = int64_t(m.rows) * per_row;
  if (int64_t(blockIdx.x) * (kThreads * 4) >= total) return;
  if (blockIdx.x == 0 && threadIdx.x == 0) *m.counter = 0;
  double sum = 0.0;
  for (int i = threadIdx.x; i < m.n_partials; i += kThreads) sum += m.partials[i];
  const float scale = scale_of(block_sum_all(sum, red), eps);
  const typename Source::View v = src.view(blockIdx.y);
  const bool vec = v.aligned() && (m.cols & 7) == 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t k = int64_t(blockIdx.x) * (kThreads * 4) + u * kThreads + threadIdx.x;
    if (k < total) load_group(m, v, vec, scale, per_row, k);
  }
}

// The same for matrices of at most kWholeElems elements, a CTA each, square sums and momentum included.
template <class Source>
__global__ void __launch_bounds__(kWholeThreads)
    whole_kernel(const __grid_constant__ Source src, double eps, uint32_t* error) {
  __shared__ double red[kWholeThreads / 32];
  grid_launch_dependents();
  const Target m = src.target(blockIdx.x);
  const typename Source::View v = src.view(blockIdx.x);
  if (threadIdx.x == 0) {
    *m.counter = 0;
    if (blockIdx.x == 0 && error != nullptr) *error = 0;
  }
  const int numel = int(m.rows * m.cols);
  const bool flat = v.aligned();
  double acc = 0.0;
  if (flat) {
    for (int k = threadIdx.x * 8; k < numel; k += kWholeThreads * 8) {
      if (k + 8 <= numel) {
        float x[8];
        v.first_eight(k, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) add_square(acc, x[i]);
      } else {
        for (int i = k; i < numel; ++i) add_square(acc, v.first_one(i));
      }
    }
  } else {
    for (int k = threadIdx.x; k < numel; k += kWholeThreads) add_square(acc, v.first_one(k));
  }
  const float scale = scale_of(block_sum_all<kWholeThreads>(acc, red), eps);  // (and a barrier: momenta are written)
  const uint32_t per_row = m.ld >> 3;
  const int total = int(m.rows * per_row);
  const bool vec = flat && (m.cols & 7) == 0;
  for (int k = threadIdx.x; k < total; k += kWholeThreads) load_group(m, v, vec, scale, per_row, k);
}

// The orthogonalised matrices as bf16 (`rounded`: which they are; NaN if a wait of the products ran out), eight
// elements of the packed result per thread, so that odd row lengths cost unaligned loads but no narrow stores.
__global__ void __launch_bounds__(kThreads)
    store_kernel(const __half* x, Shape sh, bool rounded, int64_t total, uint16_t* out, const uint32_t* error) {
  const bool bad = *error != 0;
  const int64_t numel = sh.rows * sh.cols;
  const bool vec = (sh.cols & 7) == 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t e = ((int64_t(blockIdx.x) * 4 + u) * kThreads + threadIdx.x) * 8;
    if (e >= total) break;
    int64_t z = e / numel;
    const int64_t in = e - z * numel;
    int64_t r = in / sh.cols, c = in - r * sh.cols;
    const __half* p = x + z * sh.plane + r * sh.ld + c;
    uint32_t b[4];
    if (vec) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      b[0] = w.x, b[1] = w.y, b[2] = w.z, b[3] = w.w;
    } else {
      uint16_t h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[i] = e + i < total ? __half_as_ushort(*p) : uint16_t(0);
        ++p;
        if (++c == sh.cols) {
          c = 0;
          if (++r == sh.rows) r = 0, ++z;
          p = x + z * sh.plane + r * sh.ld;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = uint32_t(h[2 * i]) | (uint32_t(h[2 * i + 1]) << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[i]));
      b[i] = bad       ? 0x7fff7fffu
             : rounded ? b[i]
                       : uint32_t(Elem<HA_BF16>::narrow(f.x * (1.0f / kScaleX))) |
                       (uint32_t(Elem<HA_BF16>::narrow(f.y * (1.0f / kScaleX))) << 16);
    }
    if (e + 8 <= total && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
      *reinterpret_cast<uint4*>(out + e) = make_uint4(b[0], b[1], b[2], b[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e + i < total) out[e + i] = uint16_t(b[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// W <- W * decay + neg_lr * O, the copy of W in DT, and the peers' copies.  neg_lr holds the shape's
// factor and the plane's scale.  The stores follow adamw_kernel's (changed sectors only with DELTA).
template <int DT, bool PEERS, bool DELTA>
__global__ void __launch_bounds__(kThreads)
    apply_kernel(const __grid_constant__ Slice s, int use_decay, Peers peers, unsigned long long* changed,
                 const uint32_t* error, uint32_t* status) {
  static_assert(!(DELTA && DT == HA_F32), "fp32 parameters are their own masters: always written");
  __shared__ uint32_t stored_in_cta;
  if (*error != 0) {  // a wait of the products ran out: the weights stay as they are
    if (threadIdx.x == 0 && status != nullptr) {
      *static_cast<volatile uint32_t*>(status) = 1u;
      __threadfence_system();
    }
    return;
  }
  const Entry& entry = s.e[blockIdx.y];
  const ha_tensor& t = entry.t;
  if (int64_t(blockIdx.x) * kApplyChunk >= t.numel) return;
  const __half* x = entry.hi;
  const uint32_t cols = entry.cols, ld = entry.ld;
  float* master = reinterpret_cast<float*>(t.master);
  void* param = reinterpret_cast<void*>(t.param);
  const uint64_t pushed = DT == HA_F32 ? t.master : t.param;
  const float decay = t.decay, lr = __fmul_rn(t.neg_lr, 1.0f / kScaleX);
  const int64_t begin = int64_t(blockIdx.x) * kApplyChunk, end = min(begin + kApplyChunk, t.numel);
  const bool vec = (t.master & 15) == 0 && (DT == HA_F32 || (t.param & 7) == 0);
  const bool vec_x = (cols & 3) == 0;
  uint32_t stored = 0;
  if (DELTA && threadIdx.x == 0) stored_in_cta = 0;
  auto update = [&](float w, float o) {
    if (use_decay) w = __fmul_rn(w, decay);
    return __fmaf_rn(lr, o, w);
  };
  // Row and column of an element, 32-bit from the chunk's first one on (a chunk has 2^14 elements).
  const int64_t row0 = begin / cols;
  const uint32_t col0 = uint32_t(begin - row0 * cols);
  auto place = [&](int64_t k, uint32_t& c) {
    const uint32_t at = col0 + uint32_t(k - begin), r = at / cols;
    c = at - r * cols;
    return x + (row0 + r) * ld + c;
  };
  auto one = [&](int64_t k) {
    uint32_t c;
    const float before = master[k];
    const float a = update(before, __half2float(*place(k, c)));
    master[k] = a;
    if constexpr (DT != HA_F32) {
      const uint16_t w = Elem<DT>::narrow(a);
      if (!DELTA || w != Elem<DT>::narrow(before)) {
        static_cast<uint16_t*>(param)[k] = w;
        if constexpr (PEERS) push1<DT>(peers, pushed, k, a);
        stored += DELTA;
      }
    } else if constexpr (PEERS) {
      push1<DT>(peers, pushed, k, a);
    }
  };
  if (vec) {
    constexpr int64_t kPass = int64_t(kThreads) * kGroups * 4;
    for (int64_t base = begin; base < end; base += kPass) {
      float4 ms[kGroups], o[kGroups];
      int64_t e[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        e[u] = base + 4 * (int64_t(threadIdx.x) + int64_t(u) * kThreads);
        if (e[u] + 4 <= end) {
          ms[u] = load4_f32(master, e[u]);
          uint32_t c;
          const __half* o_at = place(e[u], c);
          if (vec_x) {
            const uint2 w = *reinterpret_cast<const uint2*>(o_at);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
            o[u] = make_float4(a.x, a.y, b.x, b.y);
          } else {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = __half2float(*o_at++);
              if (++c == cols) c = 0, o_at += ld - cols;
            }
            o[u] = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        const bool full = e[u] + 4 <= end;
        uint2 w = make_uint2(0, 0);
        bool moved = false;
        if (full) {
          uint2 before = make_uint2(0, 0);
          if constexpr (DELTA) before = pack4<DT>(ms[u]);
          ms[u].x = update(ms[u].x, o[u].x);
          ms[u].y = update(ms[u].y, o[u].y);
          ms[u].z = update(ms[u].z, o[u].z);
          ms[u].w = update(ms[u].w, o[u].w);
          store4_f32(master, e[u], ms[u]);
          if constexpr (DT != HA_F32) {
            w = pack4<DT>(ms[u]);
            moved = w.x != before.x || w.y != before.y;
          } else if constexpr (PEERS) {
            push_f32x4(peers, pushed, e[u], ms[u]);
          }
        }
        if constexpr (DT != HA_F32) {
          bool store = full;
          if constexpr (DELTA) {  // the four lanes of a 32-byte sector store together
            uint32_t any = moved ? 1u : 0u;
            any |= __shfl_xor_sync(0xffffffffu, any, 1);
            any |= __shfl_xor_sync(0xffffffffu, any, 2);
            store = full && any;
          }
          if (store) {
            __stcs(reinterpret_cast<uint2*>(static_cast<uint16_t*>(param) + e[u]), w);
            if constexpr (PEERS) push_raw4(peers, pushed, e[u], w);
            stored += DELTA;
          }
        }
        if (!full) {
          for (int64_t k = e[u]; k < end; ++k) one(k);  // ragged tail of the tensor (one thread)
        }
      }
    }
  } else {
    for (int64_t k = begin + threadIdx.x; k < end; k += kThreads) one(k);
  }
  if constexpr (DELTA) {
    if (changed != nullptr) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) stored += __shfl_xor_sync(0xffffffffu, stored, o);
      __syncthreads();
      if ((threadIdx.x & 31) == 0 && stored) atomicAdd(&stored_in_cta, stored);
      __syncthreads();
      if (threadIdx.x == 0 && stored_in_cta) atomicAdd(changed, static_cast<unsigned long long>(stored_in_cta));
    }
  }
}

// ---------------------------------------------------------------- host side
constexpr int64_t kMaxSide = 1 << 24;
constexpr int64_t kMaxNumel = int64_t(1) << 33;  // padded 8-element groups are counted in 32 bits

int check_shape(const char* what, int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1 || rows > kMaxSide || cols > kMaxSide || rows * ((cols + 7) / 8 * 8) > kMaxNumel)
    return fail(HA_ERR_INVALID, "%s: matrices of %lld x %lld", what, (long long)rows, (long long)cols);
  return HA_OK;
}

// The planes hold scaled fp16, so the steps must keep singular values and factors in range.
int check_steps(const char* what, const ha_ns_params* ns) {
  if (ns == nullptr) return fail(HA_ERR_INVALID, "%s: NULL Newton-Schulz parameters", what);
  if (ns->steps < 1 || ns->steps > HA_NS_MAX_STEPS)
    return fail(HA_ERR_INVALID, "%s: %d steps (1 to %d)", what, ns->steps, HA_NS_MAX_STEPS);
  if (!(ns->eps >= 1e-30) || !(ns->eps <= 1e30))
    return fail(HA_ERR_INVALID, "%s: eps %g (1e-30 to 1e30)", what, ns->eps);
  double s = 1.0;
  for (int i = 0; i < ns->steps; ++i) {
    const float* c = ns->coef + 3 * i;
    if (!(ns_factor(c, s) <= kMaxFactor && std::fabs(c[1]) * s * s <= kMaxFactor &&
          std::fabs(c[2]) * s * s * s * s <= kMaxFactor))
      return fail(HA_ERR_INVALID, "%s: coefficients (%g, %g, %g) of step %d leave the fp16 range", what, c[0], c[1],
                  c[2], i);
    s = ns_growth(c, s);
    if (!(s <= kMaxGrowth)) return fail(HA_ERR_INVALID, "%s: step %d lets singular values grow to %g", what, i, s);
  }
  return HA_OK;
}

size_t partial_bytes(int64_t numel) {
  const int64_t chunk = chunk_for(numel);
  return size_t(((numel + chunk - 1) / chunk * 8 + 255) / 256 * 256);
}
// Workspace of a matrix: its partial sums and planes.
size_t matrix_bytes(int64_t rows, int64_t cols) {
  return size_t(ns_bytes_per_matrix(rows, cols)) + partial_bytes(rows * cols);
}

int check_workspace(const char* what, int64_t rows, int64_t cols, const void* ws, size_t bytes) {
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) != 0)
    return fail(HA_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  const size_t one = kHeader + matrix_bytes(rows, cols);
  if (bytes < one) return fail(HA_ERR_INVALID, "%s: workspace of %zu bytes; one matrix needs %zu", what, bytes, one);
  return HA_OK;
}

// Matrices of one shape in a pass through the workspace.
struct Group {
  NsBatch b;
  double* partials;
  int64_t chunk;   // elements of a partial sum
  int n_partials;
  int64_t begin;   // first entry of the caller's table
};
struct Pass {
  Group group[kNsShapes];
  NsBatch batches[kNsShapes];
  int groups = 0;
  int64_t matrices = 0;
  size_t used = kHeader;
  char* base;
  explicit Pass(void* ws) : base(static_cast<char*>(ws)) {}
  // Takes `n` matrices; the caller has checked that they fit.
  Group& add(int64_t n, int64_t rows, int64_t cols, int64_t begin) {
    Group& g = group[groups];
    g = Group{};
    g.begin = begin;
    g.chunk = chunk_for(rows * cols);
    g.n_partials = int((rows * cols + g.chunk - 1) / g.chunk);
    g.b.n = n;
    g.b.rows = rows;
    g.b.cols = cols;
    g.b.error = reinterpret_cast<uint32_t*>(base);
    g.b.counter = reinterpret_cast<uint32_t*>(base + 256) + matrices;
    g.partials = reinterpret_cast<double*>(base + used);
    ns_carve(&g.b, base + used + size_t(n) * partial_bytes(rows * cols));
    used += size_t(n) * matrix_bytes(rows, cols);
    matrices += n;
    ++groups;
    return g;
  }
  int run(const ha_ns_params& ns, cudaStream_t st) {
    for (int i = 0; i < groups; ++i) batches[i] = group[i].b;
    const int rc = ns_run(batches, groups, ns.coef, ns.steps, st);
    for (int i = 0; i < groups; ++i) group[i].b.out = batches[i].out, group[i].b.rounded = batches[i].rounded;
    return rc;
  }
};

unsigned load_grid(const NsBatch& b) {
  return unsigned((b.rows * b.ld_x + kLoadChunk - 1) / kLoadChunk);
}

template <int DT>
int orthogonalize(const void* src, void* dst, int64_t batch, int64_t rows, int64_t cols, const ha_ns_params& ns,
                  void* ws, size_t bytes, cudaStream_t st) {
  using raw = typename Elem<DT>::raw;
  const int64_t numel = rows * cols;
  int64_t cap = int64_t((bytes - kHeader) / matrix_bytes(rows, cols));
  if (cap > kMaxPass) cap = kMaxPass;
  for (int64_t i = 0; i < batch; i += cap) {
    const int64_t n = batch - i < cap ? batch - i : cap;
    Pass pass(ws);
    Group& g = pass.add(n, rows, cols, i);
    const raw* x = static_cast<const raw*>(src) + i * numel;
    const Shape sh{rows, cols, g.b.ld_x, g.b.plane_x};
    int64_t slice = kSliceBytes / (numel * int64_t(sizeof(raw)));
    if (slice < 1) slice = 1;
    for (int64_t k = 0; k < n; k += slice) {
      const unsigned m = unsigned(n - k < slice ? n - k : slice);
      double* part = g.partials + k * g.n_partials;
      const Target first{part, g.b.counter + k, g.b.hi[0] + k * sh.plane, g.b.lo + k * sh.plane, uint32_t(rows),
                         uint32_t(cols), uint32_t(sh.ld), g.n_partials};
      const PlainSource<DT> source{x + k * numel, numel, sh.plane, first};
      if (numel <= kWholeElems) {
        whole_kernel<<<m, kWholeThreads, 0, st>>>(source, ns.eps, i == 0 && k == 0 ? g.b.error : nullptr);
        continue;
      }
      square_sum_kernel<DT><<<dim3(unsigned(g.n_partials), m), kThreads, 0, st>>>(
          x + k * numel, numel, g.chunk, part, i == 0 && k == 0 ? g.b.error : nullptr);
      load_kernel<<<dim3(load_grid(g.b), m), kThreads, 0, st>>>(source, ns.eps);
    }
    // rows of 16-byte pieces: the last product stores the result itself
    uint16_t* out = static_cast<uint16_t*>(dst) + i * numel;
    g.b.bf16 = true;
    if ((cols & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) g.b.dst = out;
    int rc = check_launch("ha_orthogonalize (load)");
    if (rc == HA_OK) rc = pass.run(ns, st);
    if (rc != HA_OK) return rc;
    if (g.b.out < 0) continue;
    store_kernel<<<dim3(unsigned((n * numel + kLoadChunk - 1) / kLoadChunk)), kThreads, 0, st>>>(
        g.b.hi[g.b.out], sh, g.b.rounded, n * numel, out, g.b.error);
    rc = check_launch("ha_orthogonalize (store)");
    if (rc != HA_OK) return rc;
  }
  return HA_OK;
}

template <int DT>
void launch_apply(dim3 grid, cudaStream_t st, const Slice& s, int use_decay, bool delta, const Peers& peers,
                  unsigned long long* changed, const uint32_t* error, uint32_t* status) {
  if constexpr (DT != HA_F32) {
    if (delta) {
      if (peers.n > 0)
        apply_kernel<DT, true, true><<<grid, kThreads, 0, st>>>(s, use_decay, peers, changed, error, status);
      else
        apply_kernel<DT, false, true><<<grid, kThreads, 0, st>>>(s, use_decay, peers, changed, error, status);
      return;
    }
  }
  if (peers.n > 0)
    apply_kernel<DT, true, false><<<grid, kThreads, 0, st>>>(s, use_decay, peers, changed, error, status);
  else
    apply_kernel<DT, false, false><<<grid, kThreads, 0, st>>>(s, use_decay, peers, changed, error, status);
}

template <int DT>
int muon_step(const ha_tensor* t, const int64_t* shape, int64_t n, const MuonConst& c, const ha_ns_params& ns,
              bool delta, const Peers& peers, unsigned long long* changed, uint32_t* status, void* ws, size_t bytes,
              cudaStream_t st) {
  int64_t next = 0;  // entries looked at
  bool fresh = true;
  while (next < n) {
    // The entries of this pass: those with a gradient, as many as the workspace and a run hold; equal shapes
    // that follow one another make a group.
    Pass pass(ws);
    while (next < n && pass.groups < kNsShapes && (pass.groups + 1) * ns_stages(ns.steps) <= kNsStages) {
      const int64_t rows = shape[2 * next], cols = shape[2 * next + 1], begin = next;
      const size_t each = matrix_bytes(rows, cols);
      int64_t count = 0;
      bool full = false;
      for (; next < n && shape[2 * next] == rows && shape[2 * next + 1] == cols; ++next) {
        if (t[next].grad == 0) continue;
        full = pass.used + size_t(count + 1) * each > bytes || pass.matrices + count + 1 > kMaxPass;
        if (full) break;
        ++count;
      }
      if (count > 0) pass.add(count, rows, cols, begin);
      if (full) break;
    }
    if (pass.groups == 0) continue;
    for (int stage = 0; stage < 2; ++stage) {  // momentum and load; then, after the products, the weights
      struct Batch {
        MuonSource<DT> src;
        int m = 0;  // matrices of the launch
        int64_t bytes = 0;
        unsigned sums = 0, loads = 0, chunks = 0;
      } large, small;
      large.src.c = small.src.c = c;
      auto flush = [&](Batch& b) {
        if (b.m == 0) return HA_OK;
        uint32_t* error = fresh ? pass.group[0].b.error : nullptr;
        if (stage == 1) {
          launch_apply<DT>(dim3(b.chunks, unsigned(b.m)), st, b.src.s, c.use_decay, delta, peers, changed,
                           pass.group[0].b.error, status);
        } else if (&b == &small) {
          whole_kernel<<<unsigned(b.m), kWholeThreads, 0, st>>>(b.src, ns.eps, error);
          fresh = false;
        } else {
          momentum_kernel<DT><<<dim3(b.sums, unsigned(b.m)), kThreads, 0, st>>>(b.src.s, c, error);
          load_kernel<<<dim3(b.loads, unsigned(b.m)), kThreads, 0, st>>>(b.src, ns.eps);
          fresh = false;
        }
        b.m = 0;
        b.bytes = 0;
        b.sums = b.loads = b.chunks = 0;
        return check_launch(stage == 0 ? "ha_muon_step (momentum)" : "ha_muon_step (weights)");
      };
      for (int i = 0; i < pass.groups; ++i) {
        const Group& g = pass.group[i];
        const int64_t numel = g.b.rows * g.b.cols;
        const int64_t each = numel * (4 + int64_t(sizeof(typename Elem<DT>::raw)));
        for (int64_t k = g.begin, z = 0; z < g.b.n; ++k) {
          if (t[k].grad == 0) continue;
          Batch& b = stage == 0 && numel <= kWholeElems ? small : large;
          // full, or so much that the load kernel would no longer find it in L2
          if (b.m == kSlice || (stage == 0 && b.m > 0 && b.bytes + each > kSliceBytes))
            if (int rc = flush(b)) return rc;
          Entry& e = b.src.s.e[b.m++];
          e.t = t[k];
          e.partials = g.partials + z * g.n_partials;
          e.counter = g.b.counter + z;
          e.hi = (stage == 0 ? g.b.hi[0] : g.b.hi[g.b.out]) + z * g.b.plane_x;
          e.lo = g.b.lo + z * g.b.plane_x;
          e.rows = uint32_t(g.b.rows);
          e.cols = uint32_t(g.b.cols);
          e.ld = uint32_t(g.b.ld_x);
          e.n_partials = g.n_partials;
          e.chunk = g.chunk;
          b.bytes += each;
          if (unsigned(g.n_partials) > b.sums) b.sums = unsigned(g.n_partials);
          if (load_grid(g.b) > b.loads) b.loads = load_grid(g.b);
          const unsigned w = unsigned((numel + kApplyChunk - 1) / kApplyChunk);
          if (w > b.chunks) b.chunks = w;
          ++z;
        }
      }
      if (int rc = flush(large)) return rc;
      if (int rc = flush(small)) return rc;
      if (stage == 0)
        if (int rc = pass.run(ns, st)) return rc;
    }
  }
  return HA_OK;
}

}  // namespace
}  // namespace ha

extern "C" int ha_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols, size_t* out) {
  using namespace ha;
  if (out == nullptr) return fail(HA_ERR_INVALID, "ha_orthogonalize_workspace: NULL output");
  if (batch < 0) return fail(HA_ERR_INVALID, "ha_orthogonalize_workspace: batch %lld", (long long)batch);
  if (int rc = check_shape("ha_orthogonalize_workspace", rows, cols)) return rc;
  const int64_t n = batch < 1 ? 1 : (batch > kMaxPass ? kMaxPass : batch);
  *out = kHeader + size_t(n) * matrix_bytes(rows, cols);
  return HA_OK;
}

extern "C" int ha_orthogonalize(const void* src, int src_dtype, void* dst, int64_t batch, int64_t rows, int64_t cols,
                                const ha_ns_params* ns, void* workspace, size_t workspace_bytes, void* stream) {
  HA_NVTX_RANGE();
  using namespace ha;
  if (!valid_float_dtype(src_dtype)) return fail(HA_ERR_UNSUPPORTED, "ha_orthogonalize: dtype %d", src_dtype);
  if (batch < 0) return fail(HA_ERR_INVALID, "ha_orthogonalize: batch %lld", (long long)batch);
  if (int rc = check_shape("ha_orthogonalize", rows, cols)) return rc;
  if (int rc = check_steps("ha_orthogonalize", ns)) return rc;
  if (batch == 0) return HA_OK;
  if (src == nullptr || dst == nullptr) return fail(HA_ERR_INVALID, "ha_orthogonalize: NULL matrices");
  const uintptr_t elem = src_dtype == HA_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(src) % elem) != 0 || (reinterpret_cast<uintptr_t>(dst) & 1) != 0)
    return fail(HA_ERR_INVALID, "ha_orthogonalize: misaligned matrices");
  if (int rc = check_workspace("ha_orthogonalize", rows, cols, workspace, workspace_bytes)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (src_dtype) {
    case HA_F32: return orthogonalize<HA_F32>(src, dst, batch, rows, cols, *ns, workspace, workspace_bytes, st);
    case HA_BF16: return orthogonalize<HA_BF16>(src, dst, batch, rows, cols, *ns, workspace, workspace_bytes, st);
    default: return orthogonalize<HA_F16>(src, dst, batch, rows, cols, *ns, workspace, workspace_bytes, st);
  }
}

extern "C" int ha_muon_step(const ha_tensor* h_tensors, const int64_t* h_shapes, int64_t n, int grad_dtype,
                            const ha_muon_scalars* sc, const ha_ns_params* ns, int changed_only, const ha_peers* peers,
                            unsigned long long* d_changed_groups, uint32_t* d_status, void* workspace,
                            size_t workspace_bytes, void* stream) {
  HA_NVTX_RANGE();
  using namespace ha;
  if (!valid_float_dtype(grad_dtype)) return fail(HA_ERR_UNSUPPORTED, "ha_muon_step: grad dtype %d", grad_dtype);
  if (n < 0) return fail(HA_ERR_INVALID, "ha_muon_step: %lld tensors", (long long)n);
  if (sc == nullptr) return fail(HA_ERR_INVALID, "ha_muon_step: NULL scalars");
  if (int rc = check_steps("ha_muon_step", ns)) return rc;
  Peers q{};
  if (peers != nullptr) {
    if (peers->n < 0 || peers->n > HA_MAX_PEERS) return fail(HA_ERR_INVALID, "ha_muon_step: %d peers", peers->n);
    q.n = peers->n;
    for (int i = 0; i < peers->n; ++i) {
      if ((peers->delta[i] & 15) != 0)
        return fail(HA_ERR_INVALID, "ha_muon_step: peer %d offset not 16-byte aligned", i);
      q.delta[i] = peers->delta[i];
    }
  }
  if (n == 0) return HA_OK;
  if (h_tensors == nullptr || h_shapes == nullptr) return fail(HA_ERR_INVALID, "ha_muon_step: NULL table");
  const uint64_t elem = grad_dtype == HA_F32 ? 3 : 1;
  for (int64_t i = 0; i < n; ++i) {
    const ha_tensor& t = h_tensors[i];
    const int64_t rows = h_shapes[2 * i], cols = h_shapes[2 * i + 1];
    if (int rc = check_shape("ha_muon_step", rows, cols)) return rc;
    if (t.grad == 0) continue;
    if (t.numel != rows * cols || t.master == 0 || t.exp_avg == 0 || (grad_dtype != HA_F32 && t.param == 0))
      return fail(HA_ERR_INVALID, "ha_muon_step: entry %lld: %lld elements for %lld x %lld, or a NULL address",
                  (long long)i, (long long)t.numel, (long long)rows, (long long)cols);
    if (((t.grad | t.param) & elem) != 0 || ((t.master | t.exp_avg) & 3) != 0)
      return fail(HA_ERR_INVALID, "ha_muon_step: entry %lld: misaligned address", (long long)i);
    if (int rc = check_workspace("ha_muon_step", rows, cols, workspace, workspace_bytes)) return rc;
  }
  const MuonConst c{sc->mu, sc->one_minus_mu, sc->nesterov, sc->use_decay, sc->clip, sc->clip_mult};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool delta = changed_only != 0 && grad_dtype != HA_F32;
  switch (grad_dtype) {
    case HA_F32:
      return muon_step<HA_F32>(h_tensors, h_shapes, n, c, *ns, delta, q, d_changed_groups, d_status, workspace,
                               workspace_bytes, st);
    case HA_BF16:
      return muon_step<HA_BF16>(h_tensors, h_shapes, n, c, *ns, delta, q, d_changed_groups, d_status, workspace,
                               workspace_bytes, st);
    default:
      return muon_step<HA_F16>(h_tensors, h_shapes, n, c, *ns, delta, q, d_changed_groups, d_status, workspace,
                               workspace_bytes, st);
  }
}
