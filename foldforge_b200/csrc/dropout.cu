// Dropout from a counter-based generator: an update dropped, scaled and added to its residual in one pass.
// The mask is never stored: an element's word follows from the seed and the element's number alone, so the
// backward pass draws it again, and neither the grid nor a tensor's layout enters it.
//
// Measured on one B200 (device time, inputs past L2; a plain copy moves 6.55 TB/s):
//   512 x 512 x 128 bf16, a mask for all rows       forward 28.8 us (7.0 TB/s, part of it still in L2), backward 21.6
//   16384 x 4096 bf16, each element for itself      forward 66.7 us (6.0 TB/s), backward 67.9 (4.0)
//   8192 x 4096 fp32, each element for itself       forward 61.2 us (6.6 TB/s), backward 43.0 (6.2)
//   700 x 700 x 33 bf16, a mask for all rows        forward 30.8 us (3.2 TB/s), backward 28.7: single elements
//   1500 x 1500 x 16 bf16, a mask for all columns   forward 69 us (3.1 TB/s), backward 66: closer than 32 elements
// The generator bounds the bf16 backward pass where every element has its own word: ten rounds of two 32 x 32
// bit products for four elements. A product takes its pipe four cycles a warp (its counter: 66% busy), the
// exclusive ors, comparisons and conversions another pipe two each (62%), and 23 instructions an element
// issue in 68% of the slots. What helped there: the rounds' keys in the launch's parameters (86 -> 69 us with the
// next), a predicated addition for a selection, products that a block's threads share. Without effect or
// slower: one or four vectors a thread, blocks that loop.
#include "kernels.h"
#include "launch.cuh"
#include "mx8.cuh"

namespace ffb {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;  // elements of a vector: two of the generator's groups

// Philox4x32-10: J. Salmon, M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011.
// The rounds' keys are the launch's parameters, found on the host, so that a round is two products and two
// exclusive ors of three numbers; with DEVICE the seed is read from memory and each thread finds them.
struct Keys {
  uint32_t k[10], l[10], c, d;  // and the offset's halves
  __host__ __device__ __forceinline__ Keys(uint64_t seed, uint64_t offset)
      : c(static_cast<uint32_t>(offset)), d(static_cast<uint32_t>(offset >> 32)) {
    uint32_t a = static_cast<uint32_t>(seed), b = static_cast<uint32_t>(seed >> 32);
    for (int r = 0; r < 10; ++r) {
      k[r] = a;
      l[r] = b;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
  }
};
// the four words of elements 4 group .. 4 group + 3, the group in two halves
__device__ __forceinline__ uint4 philox(const Keys& key, uint32_t a, uint32_t b) {
  uint32_t c = key.c, d = key.d;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = static_cast<uint64_t>(a) * 0xD2511F53u, q = static_cast<uint64_t>(c) * 0xCD9E8D57u;
    a = static_cast<uint32_t>(q >> 32) ^ b ^ key.k[r];
    b = static_cast<uint32_t>(q);
    c = static_cast<uint32_t>(p >> 32) ^ d ^ key.l[r];
    d = static_cast<uint32_t>(p);
  }
  return make_uint4(a, b, c, d);
}
// element m's word of its group's
__device__ __forceinline__ uint32_t word_of(const uint4& words, uint64_t m) {
  return (m & 2) != 0 ? ((m & 1) != 0 ? words.w : words.z) : ((m & 1) != 0 ? words.y : words.x);
}
// Calls f(keys): the launch's, or those of the seed in memory
template <bool DEVICE, typename F>
__device__ __forceinline__ void with_keys(const Keys& launch, const DropoutParams& p, F&& f) {
  if constexpr (DEVICE) {
    f(Keys(p.device_seed[0], p.offset + p.device_seed[1]));
  } else {
    f(launch);
  }
}

// the words of elements 4 group .. 4 group + 7, group an even number
struct WordsOf8 {
  uint32_t w[kVec];
  __device__ __forceinline__ WordsOf8(const Keys& keys, uint32_t group_low, uint32_t group_high) {
    const uint4 lo = philox(keys, group_low, group_high), hi = philox(keys, group_low + 1, group_high);
    w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
  }
};

// VEC elements as they lie in memory. Eight fp32 values are one access of 32 bytes where they start on 32 bytes:
// as two of 16, every second one of a warp's 16 bytes, a store writes half sectors (11.5M fp32 gradients from
// bf16 16.4 us against 12.3).
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type load_vector(const T* p) {
  if constexpr (sizeof(T) * VEC == 32) {
    if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
      Words<2> v;
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v.w[0].x), "=r"(v.w[0].y), "=r"(v.w[0].z), "=r"(v.w[0].w), "=r"(v.w[1].x), "=r"(v.w[1].y), "=r"(v.w[1].z),
                     "=r"(v.w[1].w)
                   : "l"(p));
      return v;
    }
  }
  return load_raw<T, VEC>(p);
}
template <typename T>
__device__ __forceinline__ void store_vector(T* p, const Lanes<kVec>& f) {
  if constexpr (sizeof(T) == 4) {
    if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f.get(0)), "f"(f.get(1)), "f"(f.get(2)),
                   "f"(f.get(3)), "f"(f.get(4)), "f"(f.get(5)), "f"(f.get(6)), "f"(f.get(7))
                   : "memory");
      return;
    }
  }
  store_lanes<T, kVec>(p, f);
}

// One element: r + x scale where its word says so, else r, whatever x holds. The product is rounded to fp32 by itself: scale
// is 1 / (1 - p) rounded, at p = 1/4 too large by 2^-25 of itself, and an unrounded product (a fused multiply-add) carries
// that past sums that lie half way between two bf16 values: one element of 300 of a pair update then rounds to the
// other neighbour than its definition does. The instruction more costs 1.5% of 16384 x 4096 bf16, forward and backward (137
// -> 139 us); products of two elements an instruction take the bf16 rows kernel's fourth block of an SM (58 us for 57).
__device__ __forceinline__ float added(float x, uint32_t word, uint32_t threshold, float scale, float r) {
  asm("{\n\t.reg .pred p;\n\t.reg .f32 t;\n\tsetp.ge.u32 p, %2, %3;\n\tmul.rn.f32 t, %1, %4;\n\t@p add.rn.f32 %0, %0, t;\n\t}"
      : "+f"(r)
      : "f"(x), "r"(word), "r"(threshold), "f"(scale));
  return r;
}

// a vector of them, rounded once
template <typename TX, typename TO>
__device__ __forceinline__ void finish(const typename Raw<TX, kVec>::type& x, const typename Raw<TO, kVec>::type& residual,
                                       bool has_residual, const uint32_t (&w)[kVec], uint32_t threshold, float scale, TO* out) {
  const Lanes<kVec> v = widen<TX, kVec>(x), r = has_residual ? widen<TO, kVec>(residual) : Lanes<kVec>(0.f);
  Lanes<kVec> y;
#pragma unroll
  for (int j = 0; j < kVec; j += 2)
    y.p[j / 2] = f32x2(added(v.get(j), w[j], threshold, scale, r.get(j)), added(v.get(j + 1), w[j + 1], threshold, scale, r.get(j + 1)));
  store_vector<TO>(out, y);
}

// Each element with a word of its own: U vectors a thread, kThreads apart, all loaded before the first word is
// drawn. A block's groups share the counter's upper half (they start at a multiple of their number), so the
// first round's second product and the second round's first are the same for all of its threads.
template <typename TX, typename TO, int U, bool DEVICE>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const DropoutParams p, const __grid_constant__ Keys launch_keys, uint32_t threshold, int64_t total) {
  constexpr int kBlock = kThreads * U;  // vectors
  const int64_t base = blockIdx.x * static_cast<int64_t>(kBlock), left = total / kVec - base;
  const int n = left < kBlock ? static_cast<int>(left) : kBlock;
  const TX* x = static_cast<const TX*>(p.x) + base * kVec;
  const TO* residual = p.residual != nullptr ? static_cast<const TO*>(p.residual) + base * kVec : nullptr;
  TO* out = static_cast<TO*>(p.out) + base * kVec;
  typename Raw<TX, kVec>::type vx[U];
  typename Raw<TO, kVec>::type vr[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int v = threadIdx.x + u * kThreads;
    if (v < n) {
      vx[u] = load_vector<TX, kVec>(x + v * kVec);
      if (residual != nullptr) vr[u] = load_vector<TO, kVec>(residual + v * kVec);
    }
  }
  with_keys<DEVICE>(launch_keys, p, [&](const Keys& keys) {
    const uint64_t group = 2 * static_cast<uint64_t>(base);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = threadIdx.x + u * kThreads;
      if (v > n) continue;
      const WordsOf8 words(keys, static_cast<uint32_t>(group) + 2 * v, static_cast<uint32_t>(group >> 32));
      if (v < n) {
        finish<TX, TO>(vx[u], vr[u], residual != nullptr, words.w, threshold, p.scale, out + v * kVec);
      } else {  // the elements that do not fill a vector
#pragma unroll
        for (int j = 0; j < kVec - 1; ++j) {
          if (j >= static_cast<int>(total % kVec)) break;
          const float r = residual != nullptr ? static_cast<float>(residual[v * kVec + j]) : 0.f;
          out[v * kVec + j] = static_cast<TO>(added(static_cast<float>(x[v * kVec + j]), words.w[j], threshold, p.scale, r));
        }
      }
    }
  });
}

// A mask shared by `shared` rows, a thread in kRows of them at one place: VEC elements (a whole vector, or one
// element where rows are not whole vectors or start anywhere), whose words it draws once.
template <int VEC>
constexpr int kRowsOf = VEC == 1 ? 8 : 4;
template <typename TX, typename TO, int VEC, bool DEVICE>
__global__ void __launch_bounds__(kThreads)
    dropout_rows_kernel(const DropoutParams p, const __grid_constant__ Keys launch_keys, uint32_t threshold, uint32_t total,
                        Divisor places, Divisor chunks) {
  constexpr int kRows = kRowsOf<VEC>;
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= total) return;
  const uint32_t line = places.quotient(id), place = id - line * places.d;
  const uint32_t outer = chunks.quotient(line), chunk = line - outer * chunks.d;
  const int64_t row0 = static_cast<int64_t>(chunk) * kRows;
  const int64_t at = (outer * p.shared + row0) * p.inner + static_cast<int64_t>(place) * VEC;
  const TX* x = static_cast<const TX*>(p.x) + at;
  const TO* residual = p.residual != nullptr ? static_cast<const TO*>(p.residual) + at : nullptr;
  TO* out = static_cast<TO*>(p.out) + at;
  typename Raw<TX, VEC>::type vx[kRows];
  typename Raw<TO, VEC>::type vr[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (row0 + r < p.shared) {
      vx[r] = load_vector<TX, VEC>(x + r * p.inner);
      if (residual != nullptr) vr[r] = load_vector<TO, VEC>(residual + r * p.inner);
    }
  with_keys<DEVICE>(launch_keys, p, [&](const Keys& keys) {
    if constexpr (VEC == kVec) {
      const uint64_t group = 2 * (static_cast<uint64_t>(outer) * places.d + place);
      const WordsOf8 words(keys, static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32));
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (row0 + r < p.shared)
          finish<TX, TO>(vx[r], vr[r], residual != nullptr, words.w, threshold, p.scale, out + r * p.inner);
    } else {
      const uint64_t m = static_cast<uint64_t>(outer) * places.d + place;
      const uint32_t word = word_of(philox(keys, static_cast<uint32_t>(m >> 2), static_cast<uint32_t>(m >> 34)), m);
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (row0 + r < p.shared)
          out[r * p.inner] = static_cast<TO>(added(static_cast<float>(vx[r]), word, threshold, p.scale,
                                                   residual != nullptr ? static_cast<float>(vr[r]) : 0.f));
    }
  });
}

// Any sizes and any alignment: eight elements side by side in memory a thread, each with its own place in the
// mask; words are drawn again where an element's group is not the one before's. VECTOR: the tensors start on
// 16 bytes. Numbers of elements are Index wide.
template <typename TX, typename TO, bool VECTOR, bool DEVICE, typename Index>
__global__ void __launch_bounds__(kThreads)
    dropout_any_kernel(const DropoutParams p, const __grid_constant__ Keys launch_keys, uint32_t threshold, int64_t total) {
  const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) * kVec;
  if (first >= total) return;
  const TX* x = static_cast<const TX*>(p.x) + first;
  const TO* residual = p.residual != nullptr ? static_cast<const TO*>(p.residual) + first : nullptr;
  TO* out = static_cast<TO*>(p.out) + first;
  const int n = total - first < kVec ? static_cast<int>(total - first) : kVec;
  const Index inner = static_cast<Index>(p.inner), shared = static_cast<Index>(p.shared);
  Index row = static_cast<Index>(first) / inner;  // of the rows of all outer places
  Index column = static_cast<Index>(first) - row * inner, outer = row / shared;
  row -= outer * shared;
  uint64_t group = ~uint64_t(0);
  uint4 words = make_uint4(0, 0, 0, 0);
  uint32_t w[kVec];
  with_keys<DEVICE>(launch_keys, p, [&](const Keys& keys) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const Index m = outer * inner + column;
      if (m / 4 != group) {
        group = m / 4;
        words = philox(keys, static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32));
      }
      w[j] = word_of(words, m);
      if (++column == inner) {
        column = 0;
        if (++row == shared) {
          row = 0;
          ++outer;
        }
      }
    }
  });
  if (VECTOR && n == kVec) {
    typename Raw<TO, kVec>::type vr;
    if (residual != nullptr) vr = load_vector<TO, kVec>(residual);
    finish<TX, TO>(load_vector<TX, kVec>(x), vr, residual != nullptr, w, threshold, p.scale, out);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      if (j >= n) break;
      const float r = residual != nullptr ? static_cast<float>(residual[j]) : 0.f;
      out[j] = static_cast<TO>(added(static_cast<float>(x[j]), w[j], threshold, p.scale, r));
    }
  }
}

// all elements dropped: the residual, or zeros
template <typename TO>
__global__ void __launch_bounds__(kThreads) dropped_kernel(const TO* residual, TO* out, int64_t total) {
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads)
    out[i] = residual != nullptr ? residual[i] : static_cast<TO>(0.f);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
unsigned blocks(int64_t threads) { return static_cast<unsigned>((threads + kThreads - 1) / kThreads); }

template <typename TX, typename TO, bool DEVICE>
int dropout(const DropoutParams& p, cudaStream_t stream) {
  const int64_t total = p.outer * p.shared * p.inner;
  if (p.threshold >> 32 != 0) {
    const int64_t grid = (total + kThreads - 1) / kThreads, most = 148 * 16;
    dropped_kernel<TO><<<static_cast<unsigned>(grid < most ? grid : most), kThreads, 0, stream>>>(
        static_cast<const TO*>(p.residual), static_cast<TO*>(p.out), total);
    return static_cast<int>(cudaGetLastError());
  }
  const uint32_t threshold = static_cast<uint32_t>(p.threshold);
  const Keys keys(p.seed, p.offset);
  const bool vector = aligned(p.x) && aligned(p.residual) && aligned(p.out);
  if (vector && p.shared == 1) {
constexpr int U = 2;
    dropout_kernel<TX, TO, U, DEVICE><<<blocks((total / kVec + U) / U), kThreads, 0, stream>>>(p, keys, threshold, total);
    return static_cast<int>(cudaGetLastError());
  }
  if (p.shared > 1 && p.inner >= 32) {
    const bool whole = vector && p.inner % kVec == 0;
    const int64_t places = whole ? p.inner / kVec : p.inner, rows = whole ? kRowsOf<kVec> : kRowsOf<1>,
                  chunks = (p.shared + rows - 1) / rows;
    const int64_t most = (int64_t(1) << 31) - 1;
    if (places <= most && chunks <= most && p.outer <= most / places / chunks) {
      const int64_t items = p.outer * places * chunks;
      auto kernel = whole ? dropout_rows_kernel<TX, TO, kVec, DEVICE> : dropout_rows_kernel<TX, TO, 1, DEVICE>;
      kernel<<<blocks(items), kThreads, 0, stream>>>(p, keys, threshold, static_cast<uint32_t>(items),
                                                     Divisor(static_cast<uint32_t>(places)), Divisor(static_cast<uint32_t>(chunks)));
      return static_cast<int>(cudaGetLastError());
    }
  }
  const bool wide = total >= (int64_t(1) << 31);
  auto kernel = vector ? (wide ? dropout_any_kernel<TX, TO, true, DEVICE, uint64_t> : dropout_any_kernel<TX, TO, true, DEVICE, uint32_t>)
                       : (wide ? dropout_any_kernel<TX, TO, false, DEVICE, uint64_t> : dropout_any_kernel<TX, TO, false, DEVICE, uint32_t>);
  kernel<<<blocks((total + kVec - 1) / kVec), kThreads, 0, stream>>>(p, keys, threshold, total);
  return static_cast<int>(cudaGetLastError());
}

template <typename TX, typename TO>
int dropout(const DropoutParams& p, cudaStream_t stream) {
  return p.device_seed != nullptr ? dropout<TX, TO, true>(p, stream) : dropout<TX, TO, false>(p, stream);
}

}  // namespace

int launch_dropout(const DropoutParams& p, int x_is_f32, int out_is_f32, cudaStream_t stream) {
  if (x_is_f32) return out_is_f32 ? dropout<float, float>(p, stream) : dropout<float, __nv_bfloat16>(p, stream);
  return out_is_f32 ? dropout<__nv_bfloat16, float>(p, stream) : dropout<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

}  // namespace ffb
