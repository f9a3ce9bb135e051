// The loss of a model that is trained to rank as a teacher does, whose best
// results (ids, scores and how many, as a search returns them) are the target:
//
//   p = softmax(s / T) over the entries with an id in [0, cols),   q = softmax(x / T) over the row
//   loss = sum over entries of p_i (log p_i - log q_id(i))
//   dx_c = g / T (q_c - sum of p_i with id(i) = c)
//
// A row without entries (or whose scores are all -inf) has loss 0 and no
// gradient; an entry of p = 0 adds nothing; a logit of -inf has q = 0, so that p
// > 0 there costs infinity.
//
// Memory bounds it: x is read and dx written once, q never stored. Rows of up
// to 128 KB stay in a workgroup's registers between the softmax' sums and dx
// (two workgroups of 1024 threads fit a CU, so that one loads while the other
// stores). That leaves a thread 64 registers, and 7 or 8 vectors of 16 bytes do
// not fit beside the rest: of 7 the compiler puts 2 to 8 registers in scratch
// memory (12 to 36 bytes a thread), of 8 up to 26 (in bf16 with the gradient and
// 1024 threads 15, 64 bytes, beside 128 of the row). Longer rows are cut into
// parts: one kernel finds each part's maximum and sum, a second joins them, and
// for dx reads x again.
//
// The gradient adds up p of each entry's id by a search of all entries, for ids
// may come twice: top^2 steps a row, which few entries hide behind the row's
// bytes and many do not. us with top 10, 50, 200 and 1000: 8192 x 1000 in bf16 17,
// 23, 82 and 3080 (the loss alone 17 with 200, 76 with 1000; torch's steps are
// faster from some 500 on); with 10, 100, 1000 and 4096: 4096 x 50000 162, 178, 920
// and 10600.
//
// f32 logits take the hardware's exp2 (off by its last place) with the product's
// rounding added, and their sums are f32: against 64 bits the loss is off by 1.5e-7 to
// 1.8e-7 of itself (64 x 1000), where torch's steps in f32 are by 1.4e-7.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "device.hpp"
#include "products.hpp"
#include "rows.hpp"

namespace pxg {
namespace {

constexpr uint64_t TOP_MAX = 4096;
constexpr int PART_THREADS = 256;
constexpr uint64_t HELD_MAX = 8192;  // vectors that a workgroup's registers hold

struct Distill {
  const void* x;
  void* dx;
  const int64_t* ids;
  const float* scores;
  const int32_t* counts;
  const float* weight;
  float* loss;
  uint64_t xs, ds, is, ss;  // row strides
  float2* sums;             // each part's maximum and sum of a row
  float* picked;            // the entries' logits, rows of top
  uint64_t rows, first;     // first: rows of the launches before this one
  int cols, top, parts;
  float c, c_low;  // log2 e / T, and what its rounding left
  float t, t_low;  // 1 / T
};

template <class T>
constexpr int EACH = 16 / sizeof(T);  // elements of a vector

template <class T>
__device__ __forceinline__ uint32_t negative_infinities() {
  if constexpr (sizeof(T) == 4) return 0xFF800000u;
  return std::is_same_v<T, _Float16> ? 0xFC00FC00u : 0xFF80FF80u;
}

// d / T * log2 e for one element of type T: exp2 of it to T's last place. In
// f32 the product's rounding would show (|d| / T * 2^-24), so it is added.
template <class T>
__device__ __forceinline__ float exp_scaled(const Distill& p, float d) {
  const float y = d * p.c;
  const float e = __builtin_amdgcn_exp2f(y);
  if constexpr (sizeof(T) == 4) {
    const float r = __builtin_fmaf(d, p.c, -y) + d * p.c_low;
    return y > -150.0f ? __builtin_fmaf(e * r, 0.69314718f, e) : e;  // -inf: 0 (and NaN stays)
  }
  return e;
}
// d / T
__device__ __forceinline__ float scaled(const Distill& p, float d) {
  const float y = d * p.t;
  return fabsf(y) < __builtin_inff() ? y + (__builtin_fmaf(d, p.t, -y) + d * p.t_low) : y;
}

// The maximum m of some elements and the sum s of exp((x - m) / T); none: -inf, 0.
struct Softmax {
  float m, s;
};
__device__ __forceinline__ float or_zero(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ Softmax joined(const Distill& p, Softmax a, Softmax b) {
  const float m = fmaxf(a.m, b.m), z = or_zero(m);
  return {m, a.s * exp_scaled<float>(p, a.m - z) + b.s * exp_scaled<float>(p, b.m - z)};
}
__device__ __forceinline__ Softmax wave_joined(const Distill& p, Softmax a) {
  float m = a.m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  float s = a.s * exp_scaled<float>(p, a.m - or_zero(m));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  return {m, s};
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// weight / T
__device__ __forceinline__ float factor(const Distill& p, uint64_t row) { return scaled(p, p.weight[row]); }

// The teacher's entries of a row, in LDS: top ids (-1: not valid), p, and logits.
struct Teacher {
  int* ids;
  float *p, *logits;
};
__device__ __forceinline__ Teacher teacher_at(char* lds, int top) {
  return {(int*)lds, (float*)lds + top, (float*)lds + 2 * top};
}
// By one wavefront: p and the sum over entries of p log p; `none` if nothing is left of it.
template <class T>
__device__ __forceinline__ float read_teacher(const Distill& p, uint64_t row, const T* x, const float* picked,
                                              const Teacher& t, bool& none) {
  const int lane = threadIdx.x & 63;
  const int count = min(max(p.counts[row], 0), p.top);
  float best = -__builtin_inff();
  for (int i = lane; i < p.top; i += 64) {
    const int64_t id = i < count ? p.ids[row * p.is + i] : -1;
    const bool valid = (uint64_t)id < (uint64_t)p.cols;
    const float s = valid ? p.scores[row * p.ss + i] : -__builtin_inff();
    t.ids[i] = valid ? (int)id : -1;
    t.logits[i] = !valid ? 0.0f : picked ? picked[i] : (float)x[id];
    t.p[i] = s;
    best = fmaxf(best, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o));
  float mass = 0.0f;
  for (int i = lane; i < p.top; i += 64)
    if (t.ids[i] >= 0) mass += exp_scaled<float>(p, t.p[i] - or_zero(best));
  mass = wave_sum(mass);
  none = mass == 0.0f;
  const float log_mass = logf(mass);
  float sum = 0.0f;
  for (int i = lane; i < p.top; i += 64) {
    const float d = t.p[i] - or_zero(best);
    const float v = t.ids[i] < 0 || none ? 0.0f : exp_scaled<float>(p, d) / mass;
    t.p[i] = v;
    if (v != 0.0f) sum += v * (scaled(p, d) - log_mass);
  }
  return wave_sum(sum);
}
// By the same wavefront: - sum over entries of p log q.
__device__ __forceinline__ float cross_entropy(const Distill& p, const Teacher& t, Softmax row) {
  const float log_sum = row.s == 0.0f ? 0.0f : logf(row.s);  // 0: all logits are -inf, as d is
  float sum = 0.0f;
  for (int i = threadIdx.x & 63; i < p.top; i += 64)
    if (t.p[i] != 0.0f) sum -= t.p[i] * (scaled(p, t.logits[i] - or_zero(row.m)) - log_sum);
  return wave_sum(sum);
}
// The gradient at the entries' ids in [lo, hi), over what is stored for the
// row: eight lanes to an entry add up p of its id.
template <class T, int THREADS>
__device__ __forceinline__ void store_entries(const Distill& p, const Teacher& t, Softmax row, float k, T* dx, int lo,
                                              int hi) {
  const int sub = threadIdx.x & 7;
  for (int i0 = 0; i0 < p.top; i0 += THREADS / 8) {
    const int i = i0 + threadIdx.x / 8, id = i < p.top ? t.ids[i] : -1;
    float sum = 0.0f;
    if (id >= lo && id < hi)
      for (int j = sub; j < p.top; j += 8) sum += t.ids[j] == id ? t.p[j] : 0.0f;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (sub == 0 && id >= lo && id < hi) {
      const float q = row.s == 0.0f ? 0.0f : exp_scaled<float>(p, t.logits[i] - or_zero(row.m)) / row.s;
      dx[id] = rounded<T>(k * (q - sum));
    }
  }
}

// Vector v of a row is its elements from v EACH - phase on, 16-byte aligned;
// the first and the last may lie across its ends.
template <class T>
__device__ __forceinline__ int phase_of(const void* row) {
  return (int)((uintptr_t)row % 16 / sizeof(T));
}
template <class T>
__device__ __forceinline__ bool is_whole(int v, int phase, int cols) {
  const int64_t at = (int64_t)v * EACH<T> - phase;
  return at >= 0 && at + EACH<T> <= cols;
}
template <class T>
__device__ __forceinline__ uint4 load_ends(const T* row, int v, int phase, int cols) {
  T x[EACH<T>];
  uint4 fill = make_uint4(negative_infinities<T>(), negative_infinities<T>(), negative_infinities<T>(),
                          negative_infinities<T>());
  __builtin_memcpy(x, &fill, 16);
  const int64_t at = (int64_t)v * EACH<T> - phase;
#pragma unroll
  for (int e = 0; e < EACH<T>; ++e)
    if (at + e >= 0 && at + e < cols) x[e] = row[at + e];
  __builtin_memcpy(&fill, x, 16);
  return fill;
}
template <class T>
__device__ __forceinline__ void unpack(uint4 raw, float (&x)[EACH<T>]) {
  T v[EACH<T>];
  __builtin_memcpy(v, &raw, 16);
#pragma unroll
  for (int e = 0; e < EACH<T>; ++e) x[e] = (float)v[e];
}
template <class T, bool ONCE = false>
__device__ __forceinline__ void store_vector(T* row, int v, int phase, int cols, bool aligned, uint4 x) {
  const int64_t at = (int64_t)v * EACH<T> - phase;
  if (aligned && at >= 0 && at + EACH<T> <= cols) {
    if constexpr (ONCE) store_once(row + at, x);
    else *reinterpret_cast<uint4*>(row + at) = x;
  } else {
    T y[EACH<T>];
    __builtin_memcpy(y, &x, 16);
#pragma unroll
    for (int e = 0; e < EACH<T>; ++e)
      if (at + e >= 0 && at + e < cols) row[at + e] = y[e];
  }
}
// 16-bit logits are bound by arithmetic as much as by memory, so there
//   - the maximum is one of whole numbers, two at a time: patterns of positive
//     values grow with them, of negative ones against them, so that the largest
//     signed one is the maximum unless all are negative; then it is the smallest
//     unsigned one;
//   - x c - M is one operation, M the rounded m c (c = log2 e / T). What M's
//     rounding left is taken out of the sum;
//   - the gradient's factor goes into the exponent, which costs 2^-17 of an
//     exponential while the factor is within 2^32 of 1, and 2^-16 at most, while
//     |M| is at most 128; beyond, and in f32, it is (x - m) c and a factor.
constexpr float FAST_MAX = 128.0f;

// Vectors that are unpacked in another pass are unpacked anew: their floats would not fit the registers.
template <int N>
__device__ __forceinline__ void keep_packed(uint4 (&raw)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
}

template <class T, int N>
__device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
  if constexpr (sizeof(T) == 4) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EACH<T>];
      unpack<T>(raw[i], x);
#pragma unroll
      for (int e = 0; e < EACH<T>; ++e) m = fmaxf(m, x[e]);
    }
    return m;
  } else {
    typedef short s2 __attribute__((ext_vector_type(2)));
    typedef unsigned short u2 __attribute__((ext_vector_type(2)));
    s2 hi = {(short)0x8000, (short)0x8000};
    u2 lo = {0xFFFF, 0xFFFF};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s2, w[e]));
        lo = __builtin_elementwise_min(lo, __builtin_bit_cast(u2, w[e]));
      }
    }
    const short h = hi[0] > hi[1] ? hi[0] : hi[1];
    const unsigned short l = lo[0] < lo[1] ? lo[0] : lo[1];
    return (float)__builtin_bit_cast(T, h >= 0 ? (unsigned short)h : l);
  }
}

// dx = f exp((x - m) / T) of a vector.
template <class T>
struct Gradient {
  float m, f, offset;
  uint32_t sign;
  bool fast;
  __device__ __forceinline__ Gradient(const Distill& p, float m_, float f_) : m(m_), f(f_) {
    const float big = m * p.c;
    fast = sizeof(T) == 2 && fabsf(big) <= FAST_MAX && fabsf(f) >= 1e-30f && fabsf(f) <= 1e30f;
    offset = __builtin_amdgcn_logf(fabsf(f)) - __builtin_fmaf(m, p.c, -big) - big;  // log2
    sign = f < 0.0f ? 0x80008000u : 0u;
  }
  template <bool FAST>
  __device__ __forceinline__ uint4 of(const Distill& p, uint4 raw) const {
    float x[EACH<T>];
    unpack<T>(raw, x);
    T y[EACH<T>];
#pragma unroll
    for (int e = 0; e < EACH<T>; ++e)
      if constexpr (FAST) y[e] = rounded<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[e], p.c, offset)));
      else y[e] = rounded<T>(exp_scaled<T>(p, x[e] - m) * f);
    uint4 w;
    __builtin_memcpy(&w, y, 16);
    if constexpr (FAST) return make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
    return f == 0.0f ? make_uint4(0, 0, 0, 0) : w;  // zeros, whatever the row holds
  }
};
template <class T, int N>
__device__ __forceinline__ Softmax softmax_of(const Distill& p, uint4 (&raw)[N], Softmax before = {-__builtin_inff(), 0.0f}) {
  const float m = fmaxf(before.m, largest<T>(raw)), z = or_zero(m), big = z * p.c;
  float s = 0.0f;
  if (sizeof(T) == 2 && fabsf(big) <= FAST_MAX) {
    keep_packed(raw);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EACH<T>];
      unpack<T>(raw[i], x);
#pragma unroll
      for (int e = 0; e < EACH<T>; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], p.c, -big));
    }
    s *= __builtin_amdgcn_exp2f(-__builtin_fmaf(z, p.c, -big));
  } else {
    keep_packed(raw);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[EACH<T>];
      unpack<T>(raw[i], x);
#pragma unroll
      for (int e = 0; e < EACH<T>; ++e) s += exp_scaled<T>(p, x[e] - z);
    }
  }
  return {m, s + before.s * exp_scaled<float>(p, before.m - z)};
}

// A workgroup's row in registers: N vectors of a thread. 4096 x 50000 in bf16
// with top 100: 180 us, 4.5 TB/s. (With rows one after another in workgroups
// that load the next while they store, whose registers leave 512 threads: 225;
// with a maximum of floats and a factor: 198, for 188 past no caches.)
template <class T, int THREADS, int N, bool GRAD>
__global__ void __launch_bounds__(THREADS, 8) distill_row(Distill p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ Softmax waves[THREADS / 64];
  __shared__ int no_teacher;
  // long rows are many bytes: past the caches (188 us without, 207 with loads alone)
  constexpr bool ONCE = THREADS == 1024;
  const uint64_t row = p.first + blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* x = (const T*)p.x + row * p.xs;
  const int phase = phase_of<T>(x), vectors = (int)(((int64_t)p.cols + phase + EACH<T> - 1) / EACH<T>);
  uint4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = i * THREADS + threadIdx.x;
    if (is_whole<T>(v, phase, p.cols)) {
      const T* from = x + ((int64_t)v * EACH<T> - phase);
      raw[i] = ONCE ? load_once(from) : *reinterpret_cast<const uint4*>(from);
    }
  }
  const Teacher t = teacher_at(lds, p.top);
  float entropy = 0.0f;
  bool none = false;
  if (wave == 0) {
    entropy = read_teacher<T>(p, row, x, nullptr, t, none);
    if (lane == 0) no_teacher = none;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = i * THREADS + threadIdx.x;
    if (!is_whole<T>(v, phase, p.cols)) raw[i] = load_ends<T>(x, v, phase, p.cols);
  }
  const Softmax mine = wave_joined(p, softmax_of<T>(p, raw));
  if (lane == 0) waves[wave] = mine;
  __syncthreads();
  const Softmax all = wave_joined(p, lane < THREADS / 64 ? waves[lane] : Softmax{-__builtin_inff(), 0.0f});
  none = no_teacher;
  if (wave == 0) {
    const float other = cross_entropy(p, t, all);
    if (lane == 0) p.loss[row] = none ? 0.0f : entropy + other;
  }
  if constexpr (GRAD) {
    T* dx = (T*)p.dx + row * p.ds;
    const bool aligned = phase_of<T>(dx) == phase;
    const float k = factor(p, row);
    const Gradient<T> gradient(p, or_zero(all.m), none || all.s == 0.0f ? 0.0f : k / all.s);
    keep_packed(raw);
    auto store = [&](auto fast) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int v = i * THREADS + threadIdx.x;
        if (v < vectors)
          store_vector<T, ONCE>(dx, v, phase, p.cols, aligned, gradient.template of<decltype(fast)::value>(p, raw[i]));
      }
    };
    if (sizeof(T) == 2 && gradient.fast) store(std::true_type{});
    else store(std::false_type{});
    if (none) return;
    __syncthreads();  // what follows is stored over it
    store_entries<T, THREADS>(p, t, all, k, dx, 0, p.cols);
  }
}

// A part of a row: its maximum and sum. A workgroup past the parts gathers the entries' logits.
template <class T>
__global__ void __launch_bounds__(PART_THREADS) distill_part(Distill p) {
  __shared__ Softmax waves[PART_THREADS / 64];
  const uint64_t row = p.first + blockIdx.x / (p.parts + 1);
  const int part = blockIdx.x % (p.parts + 1), lane = threadIdx.x & 63;
  const T* x = (const T*)p.x + row * p.xs;
  if (part == p.parts) {
    const int count = min(max(p.counts[row], 0), p.top);
    for (int i = threadIdx.x; i < count; i += PART_THREADS) {
      const int64_t id = p.ids[row * p.is + i];
      if ((uint64_t)id < (uint64_t)p.cols) p.picked[row * p.top + i] = (float)x[id];
    }
    return;
  }
  const int phase = phase_of<T>(x), vectors = (int)(((int64_t)p.cols + phase + EACH<T> - 1) / EACH<T>);
  const int lo = (int)((int64_t)vectors * part / p.parts), hi = (int)((int64_t)vectors * (part + 1) / p.parts);
  constexpr int AHEAD = 4;
  const uint32_t fill = negative_infinities<T>();
  Softmax mine{-__builtin_inff(), 0.0f};
  for (int v0 = lo + (int)threadIdx.x; v0 < hi; v0 += PART_THREADS * AHEAD) {
    uint4 raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int v = v0 + i * PART_THREADS;
      raw[i] = make_uint4(fill, fill, fill, fill);
      if (v < hi && is_whole<T>(v, phase, p.cols)) raw[i] = *reinterpret_cast<const uint4*>(x + ((int64_t)v * EACH<T> - phase));
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int v = v0 + i * PART_THREADS;
      if (v < hi && !is_whole<T>(v, phase, p.cols)) raw[i] = load_ends<T>(x, v, phase, p.cols);
    }
    mine = softmax_of<T>(p, raw, mine);
  }
  mine = wave_joined(p, mine);
  if (lane == 0) waves[threadIdx.x >> 6] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    Softmax s = waves[0];
#pragma unroll
    for (int i = 1; i < PART_THREADS / 64; ++i) s = joined(p, s, waves[i]);
    p.sums[row * p.parts + part] = make_float2(s.m, s.s);
  }
}

// The parts joined: the row's loss, and the gradient's part. Without a gradient a workgroup to a row.
template <class T, bool GRAD>
__global__ void __launch_bounds__(PART_THREADS) distill_join(Distill p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ int no_teacher;
  const uint64_t row = p.first + (GRAD ? blockIdx.x / p.parts : blockIdx.x);
  const int part = GRAD ? blockIdx.x % p.parts : 0, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (!GRAD && wave) return;  // one wavefront does it
  const T* x = (const T*)p.x + row * p.xs;
  Softmax all{-__builtin_inff(), 0.0f};
  for (int i = lane; i < p.parts; i += 64) {
    const float2 s = p.sums[row * p.parts + i];
    all = joined(p, all, Softmax{s.x, s.y});
  }
  all = wave_joined(p, all);
  const Teacher t = teacher_at(lds, p.top);
  bool none = false;
  if (wave == 0) {
    const float entropy = read_teacher<T>(p, row, x, p.picked + row * p.top, t, none);
    const float other = cross_entropy(p, t, all);
    if (lane == 0) {
      no_teacher = none;
      if (part == 0) p.loss[row] = none ? 0.0f : entropy + other;
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    none = no_teacher;
    T* dx = (T*)p.dx + row * p.ds;
    const int phase = phase_of<T>(x), vectors = (int)(((int64_t)p.cols + phase + EACH<T> - 1) / EACH<T>);
    const int lo = (int)((int64_t)vectors * part / p.parts), hi = (int)((int64_t)vectors * (part + 1) / p.parts);
    const bool aligned = phase_of<T>(dx) == phase;
    const float k = factor(p, row);
    const Gradient<T> gradient(p, or_zero(all.m), none || all.s == 0.0f ? 0.0f : k / all.s);
    constexpr int AHEAD = 4;
    for (int v0 = lo + (int)threadIdx.x; v0 < hi; v0 += PART_THREADS * AHEAD) {
      uint4 raw[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int v = v0 + i * PART_THREADS;
        if (v < hi && is_whole<T>(v, phase, p.cols)) raw[i] = *reinterpret_cast<const uint4*>(x + ((int64_t)v * EACH<T> - phase));
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int v = v0 + i * PART_THREADS;
        if (v >= hi) break;
        if (!is_whole<T>(v, phase, p.cols)) raw[i] = load_ends<T>(x, v, phase, p.cols);
        store_vector<T>(dx, v, phase, p.cols, aligned,
                        gradient.fast ? gradient.template of<true>(p, raw[i]) : gradient.template of<false>(p, raw[i]));
      }
    }
    if (none) return;
    __syncthreads();  // what follows is stored over it
    const int64_t first = (int64_t)lo * EACH<T> - phase, last = (int64_t)hi * EACH<T> - phase;
    store_entries<T, PART_THREADS>(p, t, all, k, dx, (int)std::max<int64_t>(first, 0), (int)std::min<int64_t>(last, p.cols));
  }
}

// Which kernel takes a call: a row to a workgroup of `threads` with `each`
// vectors a thread, or rows in `parts`. Measured with the gradient, us, bf16:
//   16 rows of 20000     held 9.7, in parts 14.3
//   64 of 60000               14.0,          14.5
//   8192 of 9000         by 256 threads 61, by 1024 103
//   8192 of 1000         by 64 threads 15.6, by 256 25.8; 64 rows (f32) 7.3, 5.9
// (Parts of as many rows at a time as the last cache holds until they are read
// again: 1000 rows of 200000 268, of all of them 264.)
struct DistillPlan {
  int threads, each, parts;
  uint64_t bytes;
};
DistillPlan distill_plan(int type, uint64_t rows, uint64_t cols, uint64_t top) {
  DistillPlan d{0, 0, 0, 0};
  const uint64_t each = type == PXG_F32 ? 4 : 8, vectors = (cols + 2 * each - 2) / each;  // at any alignment
  if (vectors <= HELD_MAX) {
    // small workgroups where rows are many: more of them are on their way at once
    d.threads = vectors <= 256 && rows > 1024 ? 64 : vectors <= 1024 || (vectors <= 2048 && rows > 512) ? 256 : 1024;
    d.each = (int)((vectors + d.threads - 1) / d.threads);
    return d;
  }
  // about 2048 workgroups fill the chip; parts of less than 16 KB gain nothing
  const uint64_t most = std::max<uint64_t>(1, std::min<uint64_t>(256, vectors / 1024));
  d.parts = (int)std::min(most, (2048 + rows - 1) / rows);
  d.bytes = rows * d.parts * sizeof(float2) + rows * top * 4;
  return d;
}

template <class T, bool GRAD>
void run_distill(Distill p, const DistillPlan& d, hipStream_t s) {
  const unsigned lds = (unsigned)(p.top * 12);
  auto row = [&](auto threads, auto each) {
    constexpr int THREADS = decltype(threads)::value, N = decltype(each)::value;
    constexpr uint64_t MOST = LAUNCH_ROWS / 2;  // of 1024 threads
    for (uint64_t a = 0; a < p.rows; a += MOST) {
      p.first = a;
      hipLaunchKernelGGL((distill_row<T, THREADS, N, GRAD>), dim3((unsigned)std::min(MOST, p.rows - a)), dim3(THREADS), lds,
                         s, p);
      PXG_HIP(hipGetLastError());
    }
  };
  auto of = [&](auto threads) {
    switch (d.each) {
      case 1: row(threads, std::integral_constant<int, 1>{}); break;
      case 2: row(threads, std::integral_constant<int, 2>{}); break;
      case 3: row(threads, std::integral_constant<int, 3>{}); break;
      case 4: row(threads, std::integral_constant<int, 4>{}); break;
      case 5: row(threads, std::integral_constant<int, 5>{}); break;
      case 6: row(threads, std::integral_constant<int, 6>{}); break;
      case 7: row(threads, std::integral_constant<int, 7>{}); break;
      default: row(threads, std::integral_constant<int, 8>{}); break;
    }
  };
  if (d.threads == 64) {
    if (d.each == 1) row(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (d.each == 2) row(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    else row(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  } else if (d.threads == 256) {
    of(std::integral_constant<int, 256>{});
  } else if (d.threads) {
    of(std::integral_constant<int, 1024>{});
  } else {
    const uint64_t all = p.rows;
    p.parts = d.parts;
    for (uint64_t a = 0, most = LAUNCH_ROWS / (d.parts + 1); a < all; a += most) {
      const unsigned m = (unsigned)std::min(most, all - a);
      p.first = a;
      hipLaunchKernelGGL(distill_part<T>, dim3(m * (d.parts + 1)), dim3(PART_THREADS), 0, s, p);
      PXG_HIP(hipGetLastError());
      hipLaunchKernelGGL((distill_join<T, GRAD>), dim3(GRAD ? m * d.parts : m), dim3(GRAD ? PART_THREADS : 64), lds, s, p);
      PXG_HIP(hipGetLastError());
    }
  }
}

int distill(const pxg_distill* arguments, bool grad, void* stream) {
  return guard([&] {
    const pxg_distill& a = check_arguments(arguments);
    check_type(a.type, true);
    check_size("cols", a.cols);
    if (a.top == 0 || a.top > TOP_MAX) config_error("top", a.top, "must be between 1 and 4096");
    if (!(a.temperature >= 1e-6 && a.temperature <= 1e6)) config_error("temperature", 0, "must be between 1e-6 and 1e6");
    check_rows(a.type, "logits", a.logits, a.rows, a.cols, a.logits_stride);
    check_rows(PXG_F32, "ids", a.ids, a.rows, a.top, a.ids_stride);
    check_aligned("ids", a.ids, 8);
    check_rows(PXG_F32, "scores", a.scores, a.rows, a.top, a.scores_stride);
    check_rows(PXG_F32, "counts", a.counts, a.rows, 1, 1);
    check_rows(PXG_F32, "loss", a.loss, a.rows, 1, 1);
    if (grad) {
      check_rows(PXG_F32, "weight", a.weight, a.rows, 1, 1);
      check_rows(a.type, "dx", a.dx, a.rows, a.cols, a.dx_stride);
    }
    if (a.rows == 0) return;
    const DistillPlan d = distill_plan(a.type, a.rows, a.cols, a.top);
    check_aligned("workspace", a.workspace, 16);
    if (d.bytes && (!a.workspace || a.workspace_bytes < d.bytes))
      config_error("workspace_bytes", a.workspace_bytes, "must be what pxg_distill_workspace says");
    Distill p{};
    p.x = a.logits;
    p.dx = a.dx;
    p.ids = a.ids;
    p.scores = a.scores;
    p.counts = a.counts;
    p.weight = a.weight;
    p.loss = a.loss;
    p.xs = a.logits_stride;
    p.ds = a.dx_stride;
    p.is = a.ids_stride;
    p.ss = a.scores_stride;
    p.sums = (float2*)a.workspace;
    p.picked = (float*)((char*)a.workspace + a.rows * d.parts * sizeof(float2));
    p.rows = a.rows;
    p.cols = (int)a.cols;
    p.top = (int)a.top;
    const double c = 1.4426950408889634 / a.temperature, t = 1.0 / a.temperature;
    p.c = (float)c;
    p.c_low = (float)(c - p.c);
    p.t = (float)t;
    p.t_low = (float)(t - p.t);
    auto run = [&](auto kind) {
      using T = decltype(kind);
      if (grad) run_distill<T, true>(p, d, (hipStream_t)stream);
      else run_distill<T, false>(p, d, (hipStream_t)stream);
    };
    if (a.type == PXG_F32) run(float{});
    else if (a.type == PXG_F16) run((_Float16)0);
    else run((__bf16)0.0f);
  });
}

}  // namespace
}  // namespace pxg

using namespace pxg;

extern "C" {

uint64_t pxg_distill_workspace(int type, uint64_t rows, uint64_t cols, uint64_t top) {
  if (rows == 0 || rows > PRODUCT_SIZE_MAX || cols == 0 || cols > PRODUCT_SIZE_MAX || top == 0 || top > TOP_MAX) return 0;
  return distill_plan(type, rows, cols, top).bytes;
}

int pxg_distill_loss_device(const pxg_distill* a, void* stream) { return distill(a, false, stream); }
int pxg_distill_loss_grad_device(const pxg_distill* a, void* stream) { return distill(a, true, stream); }

}  // extern "C"
