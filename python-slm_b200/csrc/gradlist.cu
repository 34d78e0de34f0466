// Kernels over gradient lists: tensors that lie where the backward pass left
// them, in f32, bf16 or f16, contiguous or as rows with a pitch.
//
//   list_norm_kernel        -- one block per unit: squares, the unit's f64 partial
//                              and largest magnitude.
//   list_finalize_kernel    -- norm, clip scale, non-finite flag; the tensors' own.
//   list_clip_kernel        -- one block per unit: unscale, clip, write.
//   list_small_kernel       -- norm, clip or the step's decision of a small list.
//   list_accumulate_kernel, list_accumulate_norm_kernel -- into the flat f32
//                              accumulator (and the partials of the sums, for the
//                              last micro-batch).
//   list_decide_kernel, list_update_kernel -- the optimizer step on a list.
//
// All of them stream; nothing is a contraction, so no tensor cores.  What each is
// bound by and measured stands at the kernel.  The kernels of one call are
// chained by programmatic dependent launch: each lets the next one become
// resident at once and the next one waits for its results (pdl_wait) after it
// has issued what loads do not depend on them.  The first kernel of a call waits
// before it reads or writes anything that another call may have written, and
// triggers only then, so what the kernels behind it in the call read ahead of
// their own waits (gradients, state, unit records) was complete and visible
// already.  Those behind it (finalize, decide) may therefore trigger at once;
// whatever comes behind a call starts with a wait again, or is launched without
// the attribute (the update pass).
#include "step_device.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace slmopt {
namespace {

constexpr uint32_t kListThreads = 256;  // of one unit

// The thread's index among a unit's 256 (a block may work on several units).
__device__ __forceinline__ uint32_t unit_thread() { return threadIdx.x % kListThreads; }

// ---- L2 priorities ---------------------------------------------------------------
// What a kernel reads or writes for the last time leaves the L2 first; what the
// clip reads again soon (the list's end, see GradListView::keep) stays longest.
__device__ __forceinline__ uint64_t l2_first_out() {
  uint64_t r;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(r));
  return r;
}
__device__ __forceinline__ uint64_t l2_normal() {
  uint64_t r;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(r));
  return r;
}

// ---- element types ------------------------------------------------------------
template <uint32_t T>
constexpr uint32_t kSize = T == kGradF32 ? 4u : 2u;
template <uint32_t T>
constexpr uint32_t kVecBytes = kVec * kSize<T>;  // a vector: 32 or 16 bytes, one load
__device__ __forceinline__ uint32_t elem_bytes(uint32_t type) { return type == kGradF32 ? 4u : 2u; }

template <uint32_t T>
__device__ __forceinline__ float from_bits(uint32_t b) {
  if constexpr (T == kGradF32)
    return __uint_as_float(b);
  else if constexpr (T == kGradBf16)
    return __uint_as_float(b << 16);
  else
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
}
// Bits of element i.
template <uint32_t T>
__device__ __forceinline__ uint32_t elem_bits(const void* p, uint64_t i) {
  if constexpr (T == kGradF32)
    return static_cast<const uint32_t*>(p)[i];
  else
    return static_cast<const uint16_t*>(p)[i];
}

// 8 elements as they lie in memory, kept packed while loads are in flight.
template <uint32_t T>
struct Raw {
  static constexpr uint32_t kWords = kVecBytes<T> / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) w[i] = 0u;
  }
  // One load of a vector on its own size's boundary.
  __device__ __forceinline__ void load(const void* p, uint64_t policy) {
    if constexpr (T == kGradF32) {
      asm volatile(
          "ld.global.L1::no_allocate.L2::cache_hint.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8], %9;"
          : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
            "=r"(w[7])
          : "l"(p), "l"(policy)
          : "memory");
    } else {
      asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.b32 {%0,%1,%2,%3}, [%4], %5;"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(p), "l"(policy)
                   : "memory");
    }
  }
  // A vector at any element's address: the 16-byte blocks that hold it (the
  // neighbouring threads read the same blocks: L1), and its words shifted out.
  // The caller makes sure that the blocks lie within the tensor.
  __device__ __forceinline__ void load_shifted(const uint8_t* p) {
    const uint32_t d = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint4* block = reinterpret_cast<const uint4*>(p - d);
    constexpr uint32_t kBlocks = kWords / 4 + 1;
    uint32_t b[kBlocks * 4];
#pragma unroll
    for (uint32_t i = 0; i < kBlocks; ++i) {
      const uint4 r = block[i];
      b[4 * i] = r.x;
      b[4 * i + 1] = r.y;
      b[4 * i + 2] = r.z;
      b[4 * i + 3] = r.w;
    }
    // d bytes = (d / 8) pairs of words, (d / 4) % 2 words, (d / 2) % 2 halves.
    if (d & 8u) {
#pragma unroll
      for (uint32_t i = 0; i < kWords + 2; ++i) b[i] = b[i + 2 < kBlocks * 4 ? i + 2 : i];
    }
    if (d & 4u) {
#pragma unroll
      for (uint32_t i = 0; i < kWords + 1; ++i) b[i] = b[i + 1];
    }
    const uint32_t bits = (d & 2u) * 8u;
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i)
      w[i] = T == kGradF32 ? b[i] : __funnelshift_r(b[i], b[i + 1], bits);
  }
  // The same from a 16-byte boundary on, with the shift's whole words known to the
  // compiler (one for a contiguous unit) and its half word in bits: only what is
  // needed of the last block is loaded.
  template <uint32_t kShift>
  __device__ __forceinline__ void load_shifted_by(const uint8_t* block, uint32_t bits) {
    uint32_t b[kWords + 4];
#pragma unroll
    for (uint32_t i = 0; i < kWords / 4; ++i) {
      const uint4 r = reinterpret_cast<const uint4*>(block)[i];
      b[4 * i] = r.x;
      b[4 * i + 1] = r.y;
      b[4 * i + 2] = r.z;
      b[4 * i + 3] = r.w;
    }
    constexpr uint32_t kMore = kShift + (T == kGradF32 ? 0u : 1u);  // words of the last block
    const uint8_t* last = block + kWords * 4;
    if constexpr (kMore == 1u) {
      b[kWords] = *reinterpret_cast<const uint32_t*>(last);
    } else if constexpr (kMore == 2u) {
      const uint2 r = *reinterpret_cast<const uint2*>(last);
      b[kWords] = r.x;
      b[kWords + 1] = r.y;
    } else if constexpr (kMore > 2u) {
      const uint4 r = *reinterpret_cast<const uint4*>(last);
      b[kWords] = r.x;
      b[kWords + 1] = r.y;
      b[kWords + 2] = r.z;
      b[kWords + 3] = r.w;
    }
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
      if constexpr (T == kGradF32)
        w[i] = b[i + kShift];
      else
        w[i] = __funnelshift_r(b[i + kShift], b[i + kShift + 1], bits);
    }
  }
  // Elements from `split` on (1..7) from another vector.
  __device__ __forceinline__ void merge(const Raw& b, uint32_t split) {
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
      if constexpr (T == kGradF32) {
        if (i >= split) w[i] = b.w[i];
      } else {
        const uint32_t low = 2u * i < split ? 0xffffu : 0u;
        const uint32_t keep = 2u * i + 1u < split ? low | 0xffff0000u : low;
        w[i] = (w[i] & keep) | (b.w[i] & ~keep);
      }
    }
  }
  __device__ __forceinline__ void set(uint32_t j, uint32_t bits) {
    if constexpr (T == kGradF32)
      w[j] = bits;
    else
      w[j / 2] = (j & 1u) ? (w[j / 2] & 0xffffu) | (bits << 16) : (w[j / 2] & 0xffff0000u) | bits;
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    if constexpr (T == kGradF32) {
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
    } else if constexpr (T == kGradBf16) {
      unpack_bf16x8(make_uint4(w[0], w[1], w[2], w[3]), x);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        __half2 h;
        *reinterpret_cast<uint32_t*>(&h) = w[i];
        const float2 f = __half22float2(h);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  // Largest magnitude so far (16-bit types: in two lanes): without their sign,
  // finite values, infinity and NaN order as integers.
  __device__ __forceinline__ void top(uint32_t& m) const {
    if constexpr (T == kGradF32) {
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) m = max(m, w[j] & 0x7fffffffu);
    } else {
      m = __vimax3_u16x2(m, w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu);
      m = __vimax3_u16x2(m, w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu);
    }
  }
};

// Calls f with the whole words of the shift of a contiguous run at p, as a constant.
template <typename F>
__device__ __forceinline__ void by_shift(const uint8_t* p, F f) {
  switch ((reinterpret_cast<uintptr_t>(p) & 15u) / 4u) {
    case 0: return f(std::integral_constant<uint32_t, 0>());
    case 1: return f(std::integral_constant<uint32_t, 1>());
    case 2: return f(std::integral_constant<uint32_t, 2>());
    default: return f(std::integral_constant<uint32_t, 3>());
  }
}

// A thread's largest magnitude as f32 bits.
template <uint32_t T>
__device__ __forceinline__ uint32_t top_f32(uint32_t m) {
  if constexpr (T == kGradF32)
    return m;
  else
    return __float_as_uint(from_bits<T>(max(m & 0xffffu, m >> 16))) & 0x7fffffffu;
}

// ---- where a unit's elements lie -------------------------------------------------
// A thread's place in a unit, moved from vector to vector (256 vectors apart)
// without a division: the row-major position is kept as an address and a column.
// A contiguous unit is one row.
template <uint32_t T>
struct Rows {
  uint8_t* p;         // the next element
  uint32_t col;       // its column
  uint32_t columns;
  uint32_t col_step;  // of 2,048 elements
  uint64_t step;      // bytes, before a wrap
  uint64_t wrap;      // bytes from a row's end to the next row
  // At element e of the unit.
  __device__ __forceinline__ Rows(const GradUnit& u, uint32_t e) {
    p = static_cast<uint8_t*>(const_cast<void*>(u.ptr));
    if (u.flags & kGradPitched) {
      columns = u.columns;
      const uint32_t k = u.column + e;
      const uint32_t row = k / columns;
      col = k - row * columns;
      p += (int64_t(row * u.row_stride) + col - u.column) * int64_t(kSize<T>);
      const uint32_t rows = kListThreads * kVec / columns;
      col_step = kListThreads * kVec - rows * columns;
      step = (rows * u.row_stride + col_step) * kSize<T>;
      wrap = (u.row_stride - columns) * kSize<T>;
    } else {
      columns = u.count;
      col = e;
      p += uint64_t(e) * kSize<T>;
      col_step = kListThreads * kVec;
      step = uint64_t(col_step) * kSize<T>;
      wrap = 0u;
    }
  }
  __device__ __forceinline__ void next_vector() {
    p += step;
    col += col_step;
    if (col >= columns) {
      col -= columns;
      p += wrap;
    }
  }
  __device__ __forceinline__ void next_element() {
    p += kSize<T>;
    if (++col == columns) {
      col = 0u;
      p += wrap;
    }
  }
  // Whether the next vector is one run on its boundary.
  __device__ __forceinline__ bool aligned() const {
    return col + kVec <= columns && reinterpret_cast<uintptr_t>(p) % kVecBytes<T> == 0u;
  }
  // The next n <= 8 elements, the rest zero.  inside: see inside_unit; off the
  // boundaries a vector is shifted from its blocks, and one that goes on in the
  // next row put together from two.
  __device__ __forceinline__ void load(Raw<T>& raw, uint32_t n, bool inside,
                                       uint64_t policy) const {
    if (n == kVec && aligned()) {
      raw.load(p, policy);
    } else if (n == kVec && inside && columns >= kVec) {
      raw.load_shifted(p);
      if (col + kVec > columns) {
        Raw<T> next;
        next.load_shifted(p + wrap);
        raw.merge(next, columns - col);
      }
    } else {
      raw.zero();
      Rows r = *this;
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) {
        if (j < n) {
          raw.set(j, elem_bits<T>(r.p, 0));
          r.next_element();
        }
      }
    }
  }
};
// Whether the 16-byte blocks around the 8 elements from e on lie between the
// tensor's first and last element (in memory, gaps between its rows included).
__device__ __forceinline__ bool inside_unit(const GradUnit& u, uint32_t e) {
  return (u.index > 0u || e >= kVec) && e + 2u * kVec <= u.count;
}
__device__ __forceinline__ uint32_t vector_elems(uint32_t e, uint32_t count) {
  return e >= count ? 0u : count - e < kVec ? count - e : kVec;
}

// n <= 8 elements of contiguous memory one by one, the rest zero.
template <uint32_t T>
__device__ __forceinline__ void gather_flat(Raw<T>& raw, const uint8_t* p, uint32_t n) {
  raw.zero();
#pragma unroll
  for (uint32_t j = 0; j < kVec; ++j)
    if (j < n) raw.set(j, elem_bits<T>(p, j));
}

template <bool kRows>
__device__ __forceinline__ GradUnit load_unit(const GradUnit* units, uint32_t i) {
  GradUnit u;
  const uint4* p = reinterpret_cast<const uint4*>(units + i);
  *reinterpret_cast<uint4*>(&u) = __ldg(p);
  *(reinterpret_cast<uint4*>(&u) + 1) = __ldg(p + 1);
  if constexpr (kRows) *(reinterpret_cast<uint4*>(&u) + 2) = __ldg(p + 2);
  return u;
}

// ---- norm ----------------------------------------------------------------------
// One read of the gradients: 2 or 4 bytes an element, so DRAM should bound it; a
// first form (unscaling and squaring each value, 66 warp instructions an 8-element
// vector) was bound by issue at 71 % instead.  Squares by packed fused multiply-adds of the
// stored values take 40, 32 registers keep 8 blocks of 256 threads a SM resident
// with 64 bytes a thread on their way: 135M bf16 in 42-44 us with the finalize
// (6.5 TB/s; a kernel that only reads the same bytes takes 39.4-42.7), 49 us at
// the start.  Off the vector boundaries a vector costs two loads and a shift:
// 120M bf16 in odd-sized packed tensors 57.5 us against 37.8 (vectors start at the
// tensor's first element, not at the address's boundary: the sum's bits depend on
// the sizes alone).
// Squares are formed of the stored values times the largest power of two that is
// not above 1 / scale: at most the unscaled values and half of them at least, so
// that no square overflows that is finite in the flat norm, without a division per
// element (the product does not show: 135M bf16 at 65,536 42.5 us without it,
// 42.4 with); the finalize divides the f64 sum by the exact (scale * factor)^2.
__device__ __forceinline__ float square_factor(float scale) {
  const uint32_t bits = __float_as_uint(scale), e = bits >> 23;  // scale > 0
  if (e == 0u) return __uint_as_float(254u << 23);  // 2^127, for a subnormal scale
  const uint32_t below = (bits & 0x7fffffu) != 0u ? 1u : 0u;
  return __uint_as_float((e + below >= 254u ? 1u : 254u - e - below) << 23);  // 2^-126 at the least
}

// Two f32 operations in one instruction, each rounded alone.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The term of one 8-element vector: x0^2 + x1^2 + x2^2 + x3^2 and x4^2 + ... + x7^2
// side by side, each by a product and three fused multiply-adds, their f32 sum,
// then the lane's f64.  At most 5 roundings of non-negative terms: 5 * 2^-24
// relative.
template <bool kFactor>
__device__ __forceinline__ double add_vector(double acc, const float (&x)[8], float factor) {
  uint64_t s = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    uint64_t q = pair(x[j], x[j + 4]);
    if constexpr (kFactor) q = mul2(q, pair(factor, factor));
    s = j == 0 ? mul2(q, q) : fma2(q, q, s);
  }
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(s));
  return __dadd_rn(acc, static_cast<double>(__fadd_rn(lo, hi)));
}

// The fixed tree of one unit: thread t owns the unit's vectors t, t + 256, ...
// (elements past the end count as +0.0); the block folds as the flat norm's does.
template <uint32_t T, bool kFactor>
struct Squares {
  double acc = 0.0;
  uint32_t top = 0u;
  float factor;
  __device__ __forceinline__ void take(const Raw<T>& raw) {
    float x[8];
    raw.unpack(x);
    raw.top(top);
    acc = add_vector<kFactor>(acc, x, factor);
  }
};

template <uint32_t T, bool kFactor>
__device__ __forceinline__ void flat_squares(Squares<T, kFactor>& sq, const uint8_t* base,
                                             uint32_t count, uint64_t policy) {
  constexpr uint32_t kBatch = T == kGradF32 ? 2 : 4;  // 64 bytes of loads per thread in flight
  constexpr uint32_t kStep = kListThreads * kVecBytes<T>;
  const uint32_t whole = count / kVec;
  uint32_t v = unit_thread();
  if (reinterpret_cast<uintptr_t>(base) % kVecBytes<T> == 0u) {
    const uint8_t* p = base + v * kVecBytes<T>;
    for (; v + (kBatch - 1) * kListThreads < whole; v += kBatch * kListThreads) {
      Raw<T> raw[kBatch];
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) raw[b].load(p + b * kStep, policy);
      p += kBatch * kStep;
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) sq.take(raw[b]);
    }
    for (; v < whole; v += kListThreads, p += kStep) {
      Raw<T> raw;
      raw.load(p, policy);
      sq.take(raw);
    }
  } else {
    // Off the boundaries: the first and the last vector, whose blocks can reach
    // beyond the tensor, element by element.
    const uint32_t d = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base)) & 15u;
    by_shift(base, [&](auto shift) {
      for (; v < whole; v += kListThreads) {
        Raw<T> raw;
        if (v > 0u && v + 1u < whole)
          raw.template load_shifted_by<decltype(shift)::value>(base - d + v * kVecBytes<T>,
                                                               (d & 2u) * 8u);
        else
          gather_flat(raw, base + v * kVecBytes<T>, kVec);
        sq.take(raw);
      }
    });
  }
  if (unit_thread() == whole % kListThreads && count % kVec) {
    Raw<T> raw;
    gather_flat(raw, base + whole * kVecBytes<T>, count % kVec);
    sq.take(raw);
  }
}

template <uint32_t T, bool kFactor>
__device__ __forceinline__ void row_squares(Squares<T, kFactor>& sq, const GradUnit& u,
                                            uint64_t policy) {
  const uint32_t count = u.count;
  uint32_t e = unit_thread() * kVec;
  Rows<T> rows(u, e);
  if (u.flags & kGradVector) {
    // Every vector is one aligned run.
    constexpr uint32_t kBatch = T == kGradF32 ? 2 : 4;
    for (; e < count; e += kBatch * kListThreads * kVec) {
      Raw<T> raw[kBatch];
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        if (e + b * (kListThreads * kVec) < count)
          raw[b].load(rows.p, policy);
        else
          raw[b].zero();
        rows.next_vector();
      }
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) sq.take(raw[b]);
    }
    return;
  }
  for (; e < count; e += kListThreads * kVec) {
    Raw<T> raw;
    rows.load(raw, vector_elems(e, count), inside_unit(u, e), policy);
    rows.next_vector();
    sq.take(raw);
  }
}

// kRows: the list has pitched tensors.  The kernels without them need fewer
// registers, so more of their loads are in flight.
template <uint32_t T, bool kFactor, bool kRows>
__device__ __forceinline__ double unit_squares(const GradUnit& u, const GradListView& list,
                                               float factor, uint32_t& top) {
  Squares<T, kFactor> sq;
  sq.factor = factor;
  const uint64_t policy = blockIdx.x < list.keep ? l2_first_out() : l2_normal();
  if (kRows && (u.flags & kGradPitched))
    row_squares(sq, u, policy);
  else
    flat_squares(sq, static_cast<const uint8_t*>(u.ptr), u.count, policy);
  top = top_f32<T>(sq.top);
  return sq.acc;
}

__device__ __forceinline__ double fold_warp(double v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = __dadd_rn(v, __shfl_down_sync(kFull, v, off));
  return v;
}
// The halving tree over n (a power of two) warps' sums.
template <int n>
__device__ __forceinline__ double fold_sums(const double* sums) {
  double w[n];
#pragma unroll
  for (int i = 0; i < n; ++i) w[i] = sums[i];
#pragma unroll
  for (int off = n / 2; off >= 1; off >>= 1) {
#pragma unroll
    for (int i = 0; i < off; ++i) w[i] = __dadd_rn(w[i], w[i + off]);
  }
  return w[0];
}

// Folds a unit's 256 lanes and stores the partial.  `slot` is shared memory of
// these 256 threads alone, `barrier` theirs too.
struct UnitSlot {
  double sum[kListThreads / 32];
  uint32_t top[kListThreads / 32];
};
__device__ __forceinline__ void unit_barrier(uint32_t barrier) {
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kListThreads) : "memory");
}
__device__ __forceinline__ void fold_unit(double v, uint32_t top, UnitSlot& slot,
                                          uint32_t barrier, GradPartial* to) {
  v = fold_warp(v);
  top = __reduce_max_sync(kFull, top);
  const uint32_t warp = unit_thread() / 32u;
  if ((threadIdx.x & 31u) == 0u) {
    slot.sum[warp] = v;
    slot.top[warp] = top;
  }
  unit_barrier(barrier);
  if (unit_thread() == 0u) {
#pragma unroll
    for (uint32_t i = 0; i < kListThreads / 32; ++i) top = max(top, slot.top[i]);
    const double sum = fold_sums<kListThreads / 32>(slot.sum);
    *reinterpret_cast<uint4*>(to) =
        make_uint4(uint32_t(__double2loint(sum)), uint32_t(__double2hiint(sum)), top, 0u);
  }
}

template <bool kFactor, bool kRows>
__device__ __forceinline__ double unit_squares_any(const GradUnit& u, const GradListView& list,
                                                   float factor, uint32_t& top) {
  switch (u.flags & kGradTypeMask) {
    case kGradF32:
      return unit_squares<kGradF32, kFactor, kRows>(u, list, factor, top);
    case kGradBf16:
      return unit_squares<kGradBf16, kFactor, kRows>(u, list, factor, top);
    default: return unit_squares<kGradF16, kFactor, kRows>(u, list, factor, top);
  }
}

template <bool kRows>
__device__ __forceinline__ void unit_partial(const GradListView& list, const GradUnit& u,
                                             float factor, UnitSlot& slot, uint32_t barrier,
                                             GradPartial* to) {
  uint32_t top = 0u;
  const double sum = factor == 1.0f ? unit_squares_any<false, kRows>(u, list, factor, top)
                                    : unit_squares_any<true, kRows>(u, list, factor, top);
  fold_unit(sum, top, slot, barrier, to);
}

// ---- the norm from the partials ----------------------------------------------------
// The fixed tree over a run of partials: 1,024 lanes, lane t adds partials t,
// t + 1024, ... in order; lanes fold by warps of 32, the 32 warps' sums by halves.
// kThreads threads (thread index t, a barrier of their own) hold 1,024 / kThreads
// lanes each, with at least 8 loads in flight.  Valid in thread 0.
constexpr uint32_t kLanes = 1024;
struct LaneSlot {
  double sum[kLanes / 32];
  uint32_t top[kLanes / 32];
};
template <uint32_t kThreads>
__device__ __forceinline__ void sum_partials(const GradPartial* partials, uint32_t count,
                                             uint32_t t, uint32_t barrier, LaneSlot& slot,
                                             double& sum, uint32_t& top) {
  constexpr uint32_t kHold = kLanes / kThreads;
  constexpr uint32_t kAhead = kHold < 8 ? 8 / kHold : 1;  // steps of kLanes loaded together
  double v[kHold];
  top = 0u;
#pragma unroll
  for (uint32_t h = 0; h < kHold; ++h) v[h] = 0.0;
  for (uint32_t i0 = t; i0 < count; i0 += kAhead * kLanes) {
    uint4 q[kAhead][kHold];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
#pragma unroll
      for (uint32_t h = 0; h < kHold; ++h) {
        const uint32_t i = i0 + a * kLanes + h * kThreads;
        q[a][h] = i < count ? __ldcg(reinterpret_cast<const uint4*>(partials + i))
                            : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) {
#pragma unroll
      for (uint32_t h = 0; h < kHold; ++h) {
        v[h] = __dadd_rn(v[h], __hiloint2double(int(q[a][h].y), int(q[a][h].x)));
        top = max(top, q[a][h].z);
      }
    }
  }
  top = __reduce_max_sync(kFull, top);
#pragma unroll
  for (uint32_t h = 0; h < kHold; ++h) {
    v[h] = fold_warp(v[h]);
    const uint32_t warp = (t + h * kThreads) / 32u;
    if ((t & 31u) == 0u) {
      slot.sum[warp] = v[h];
      slot.top[warp] = top;
    }
  }
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kThreads) : "memory");
  sum = 0.0;
  if (t < 32u) {
    // The halving tree over 32 sums is a shuffle tree over a warp.
    sum = fold_warp(slot.sum[t]);
    top = __reduce_max_sync(kFull, slot.top[t]);
  }
}

// The f64 sum of the unscaled squares.
__device__ __forceinline__ double unscaled_sum(double sum, float scale) {
  const double s = __dmul_rn(static_cast<double>(scale), static_cast<double>(square_factor(scale)));
  return s == 1.0 ? sum : __ddiv_rn(sum, __dmul_rn(s, s));
}
__device__ __forceinline__ float unscaled_top(uint32_t top, float scale) {
  return __fdiv_rn(__uint_as_float(top), scale);
}

__device__ __forceinline__ void write_tensor(const GradListOut& out, uint32_t t, double sum,
                                             uint32_t top, float scale, int kind) {
  const float largest = unscaled_top(top, scale);
  if (out.tensor_norms)
    out.tensor_norms[t] =
        kind != 0 ? largest : __double2float_rn(__dsqrt_rn(unscaled_sum(sum, scale)));
  if (out.tensor_max) out.tensor_max[t] = largest;
}

// The four values of a call: norm, clip scale, largest magnitude, non-finite flag.
__device__ __forceinline__ float4 norm_values(double raw, uint32_t top, float scale,
                                              float max_norm, int kind) {
  const double sum = unscaled_sum(raw, scale);
  const float largest = unscaled_top(top, scale);
  const float norm = kind != 0 ? largest : __double2float_rn(__dsqrt_rn(sum));
  // The flat step's formula: the sum rounded once to f32, f32 root and quotient.
  const float root = kind != 0 ? largest : __fsqrt_rn(__double2float_rn(sum));
  const bool bad = !finite_f32(norm) || !finite_f32(largest) || !finite_f32(root);
  float clip = 1.0f;
  if (bad)
    clip = 0.0f;
  else if (root > 0.0f)
    clip = fminf(__fdiv_rn(max_norm, root), 1.0f);
  return make_float4(norm, clip, largest, bad ? 1.0f : 0.0f);
}
__device__ __forceinline__ void write_norm(const GradListOut& out, const float4& v, double sum) {
  out.result[0] = v.x;
  out.result[1] = v.y;
  out.result[2] = v.z;
  out.result[3] = v.w;
  if (out.sum_squares) *out.sum_squares = sum;
}

// The step's decision (clip, skip, scaler).
__device__ __forceinline__ void write_step(double raw, uint32_t top, DeviceScaler* scaler,
                                           DeviceStepState* st, const FinalizeParams& fp) {
  const float scale = fp.dynamic ? scaler->scale : fp.static_scale;
  const double sum = unscaled_sum(raw, scale);
  const uint32_t nonfinite =
      !isfinite(sum) || !finite_f32(unscaled_top(top, scale)) ? 1u : 0u;
  const StepDecision d =
      decide_step(sum, nonfinite, scale, fp.dynamic ? scaler->good_steps : 0u, fp);
  write_decision(d, sum, nonfinite, scale, st, scaler, fp);
  st->result_nonfinite = 0u;
}

// scaler: where the loss scale is, if it is on the device.  The norm is finished
// by a kernel of its own: a completion counter would have to be shared by
// concurrent calls of a list, and cost more than the chained launch (4.5M
// elements: 11.9 us with the last of 1,107 blocks finishing, 8.2 us with two
// kernels).
template <bool kRows>
__global__ void __launch_bounds__(kListThreads, kRows ? 5 : 8)
    list_norm_kernel(GradListView list, float scale, const DeviceScaler* scaler,
                     GradPartial* partials) {
  __shared__ UnitSlot slot;
  // The kernels behind may start to read gradients once all blocks are here, so
  // their producers must be done by then: wait first.  A bind just ahead writes
  // the unit's record, so that is read behind the wait too.
  pdl_wait();
  pdl_trigger();
  const GradUnit u = load_unit<kRows>(list.units, blockIdx.x);
  unit_partial<kRows>(list, u, square_factor(scaler ? scaler->scale : scale), slot, 1u,
                      partials + blockIdx.x);
}

// Block 0: the list's values; every further block 8 tensors' own, 128 threads each
// (a block per tensor took its 1,024 threads' room from the norm's last blocks).
constexpr uint32_t kTensorThreads = 128, kTensorsPerBlock = kLanes / kTensorThreads;
__global__ void __launch_bounds__(kLanes)
    list_finalize_kernel(GradListView list, const GradPartial* partials, float scale,
                         float max_norm, int kind, GradListOut out) {
  __shared__ LaneSlot lanes[kTensorsPerBlock];
  pdl_trigger();
  const uint32_t group = threadIdx.x / kTensorThreads;
  const uint32_t t = (blockIdx.x - 1u) * kTensorsPerBlock + group;
  uint32_t begin = 0u, end = list.n_units;
  if (blockIdx.x > 0u) {
    if (t >= list.n_tensors) return;  // its 128 threads together
    begin = __ldg(&list.tensors[t].first_unit);
    if (t + 1u < list.n_tensors) end = __ldg(&list.tensors[t + 1u].first_unit);
  }
  pdl_wait();
  double sum;
  uint32_t top;
  if (blockIdx.x == 0u) {
    sum_partials<kLanes>(partials, end, threadIdx.x, 0u, lanes[0], sum, top);
    if (threadIdx.x == 0u)
      write_norm(out, norm_values(sum, top, scale, max_norm, kind), unscaled_sum(sum, scale));
  } else {
    const uint32_t i = threadIdx.x % kTensorThreads;
    sum_partials<kTensorThreads>(partials + begin, end - begin, i, 1u + group, lanes[group], sum,
                                 top);
    if (i == 0u) write_tensor(out, t, sum, top, scale, kind);
  }
}

// The step's decision from the partials.
__global__ void __launch_bounds__(kLanes)
    list_decide_kernel(GradListView list, const GradPartial* partials, DeviceScaler* scaler,
                       DeviceStepState* st, FinalizeParams fp) {
  __shared__ LaneSlot lanes;
  pdl_trigger();
  pdl_wait();
  double sum;
  uint32_t top;
  sum_partials<kLanes>(partials, list.n_units, threadIdx.x, 0u, lanes, sum, top);
  if (threadIdx.x == 0) write_step(sum, top, scaler, st, fp);
}

// ---- clip ----------------------------------------------------------------------
// y = round(x * (clip / scale)): a second read and the write behind the norm's
// read.  DRAM bounds it: 135M bf16 read, mostly read again (the L2 keeps the last
// 24 MB, see kGradKeepBytes) and written are 790 MB, 120 us at 6.57 TB/s; measured
// 125-129 us.  Keeping more on chip than the L2 does was not tried: 30 MB of shared
// memory would save 4.6 us.
constexpr uint32_t kNoRows = 0u, kRowVectors = 1u, kAnyRows = 2u;
template <uint32_t T>
__device__ __forceinline__ uint32_t to_bits(float y) {
  if constexpr (T == kGradF32)
    return __float_as_uint(y);
  else if constexpr (T == kGradBf16)
    return __bfloat16_as_ushort(__float2bfloat16_rn(y));
  else
    return __half_as_ushort(__float2half_rn(y));
}
// A vector on its own size's boundary; written once, so first to leave the L2.
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[4]) {
  asm volatile("st.global.L2::cache_hint.v4.b32 [%0], {%1,%2,%3,%4}, %5;" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "l"(l2_first_out())
               : "memory");
}
template <uint32_t T>
__device__ __forceinline__ void store8(void* p, const float (&y)[8]) {
  if constexpr (T == kGradF32) {
    asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p),
                 "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]),
                 "f"(y[7])
                 : "memory");
  } else {
    uint32_t w[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if constexpr (T == kGradBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    store_words(p, w);
  }
}
template <uint32_t T>
__device__ __forceinline__ void store1(void* p, uint64_t i, float y) {
  if constexpr (T == kGradF32)
    static_cast<float*>(p)[i] = y;
  else
    static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(to_bits<T>(y));
}

// The factor of the clip call, clip / scale rounded to f32: one product per
// element.  Where the quotient is no normal f32 (extreme scales) it is split
// into a normal factor and a power of two.
struct ClipFactor {
  float factor, power;
  __device__ __forceinline__ ClipFactor(float clip, float scale) {
    power = 1.0f;
    factor = __fdiv_rn(clip, scale);
    if (factor < 1.17549435e-38f && clip > 0.0f) {
      power = 5.42101086e-20f;  // 2^-64
      factor = __fdiv_rn(__fmul_rn(clip, 1.84467441e19f), scale);
    } else if (!finite_f32(factor)) {
      power = 1.84467441e19f;  // 2^64
      factor = __fdiv_rn(__fmul_rn(clip, 5.42101086e-20f), scale);
    }
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float y = __fmul_rn(x, factor);
    return power == 1.0f ? y : __fmul_rn(y, power);
  }
};

// Elements before the first vector boundary of p.
template <uint32_t T>
__device__ __forceinline__ uint32_t peel_of(const void* p, uint32_t count) {
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) % kVecBytes<T>;
  const uint32_t n = (kVecBytes<T> - off) % kVecBytes<T> / kSize<T>;
  return n < count ? n : count;
}

template <uint32_t T, uint32_t O>
__device__ __forceinline__ void clip_raw(const Raw<T>& raw, const ClipFactor& f, void* to) {
  float x[8];
  raw.unpack(x);
#pragma unroll
  for (uint32_t j = 0; j < kVec; ++j) x[j] = f(x[j]);
  store8<O>(to, x);
}

// What the clip needs of the norm, which may still be on its way: it is waited
// for once per block, after the first loads have been issued.  Lists of few units
// have no finalize kernel; every block adds the partials for itself (one launch
// and one hop less: see kGradOwnNorm).  kOwn: whether the kernel can do that.  The
// forms for contiguous tensors and for rows on the boundaries come without it as well,
// for larger lists: its registers make them spill (60M bf16 in columns in place
// 68 us without, 82 with; into bf16 69 against 72).  The form for any rows has it
// always (60M bf16 in odd columns 135 us, against 138 without).
struct ClipNorm {
  const float* result;          // of the finalize kernel, or NULL:
  const GradPartial* partials;  // what to form it from
  uint32_t count;
  float max_norm;
  int kind;
  GradListOut out;
};
template <bool kOwn>
struct ClipState {
  const ClipNorm* norm;
  float scale;
  float clip, bad;
  bool known;
  // False when a gradient is not finite, which leaves the outputs alone.  Called
  // by the whole block.
  __device__ __forceinline__ bool ready() {
    if (!known) {
      pdl_wait();
      if (!kOwn || norm->result) {
        clip = __ldcg(norm->result + 1);
        bad = __ldcg(norm->result + 3);
      } else {
        __shared__ LaneSlot lanes;
        __shared__ float2 s_clip;
        double sum;
        uint32_t top;
        sum_partials<kListThreads>(norm->partials, norm->count, threadIdx.x, 0u, lanes, sum, top);
        if (threadIdx.x == 0u) {
          const float4 v = norm_values(sum, top, scale, norm->max_norm, norm->kind);
          s_clip = make_float2(v.y, v.w);
          if (blockIdx.x == 0u) write_norm(norm->out, v, unscaled_sum(sum, scale));
        }
        __syncthreads();
        clip = s_clip.x;
        bad = s_clip.y;
      }
      known = true;
    }
    return bad == 0.0f;
  }
};

// One unit of the clip, each element read and written by the same thread.
// Contiguous on both sides: vectors start at the output's boundaries, and the
// input is shifted where it lies off them.
// kAligned: both units lie on the boundaries (kGradVector).  kShift: whether the
// input can lie off them where the output is on them (not in place).
template <uint32_t T, uint32_t O, bool kAligned, bool kShift, typename S>
__device__ __forceinline__ void clip_flat(const uint8_t* src, uint8_t* dst, uint32_t count,
                                          float scale, S& state) {
  constexpr uint32_t kBatch = T == kGradF32 ? 2 : 4;
  constexpr uint32_t kStep = kListThreads * kVecBytes<T>;
  const uint32_t peel = kAligned ? 0u : peel_of<O>(dst, count);
  const uint8_t* from = src + peel * kSize<T>;
  uint8_t* to = dst + peel * kSize<O>;
  const uint32_t whole = (count - peel) / kVec;
  uint32_t head = peel, tail = peel + whole * kVec;  // left over: [0, head), [tail, count)
  uint32_t v = unit_thread();
  if (!kShift || reinterpret_cast<uintptr_t>(from) % kVecBytes<T> == 0u) {
    const uint64_t policy = l2_first_out();
    Raw<T> raw[kBatch];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b)  // on their way while the norm is finished
      if (v + b * kListThreads < whole) raw[b].load(from + v * kVecBytes<T> + b * kStep, policy);
    if (!state.ready()) return;
    const ClipFactor f(state.clip, scale);
    while (v < whole) {
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b)
        if (v + b * kListThreads < whole)
          clip_raw<T, O>(raw[b], f, to + (v + b * kListThreads) * kVecBytes<O>);
      v += kBatch * kListThreads;
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b)
        if (v + b * kListThreads < whole) raw[b].load(from + v * kVecBytes<T> + b * kStep, policy);
    }
  } else {
    if (!state.ready()) return;
    const ClipFactor f(state.clip, scale);
    // The blocks of the first and the last vector can reach beyond the tensor.
    const uint32_t d = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) & 15u;
    by_shift(from, [&](auto shift) {
      constexpr uint32_t kShifted = T == kGradF32 ? 1 : 4;
      for (v += 1u; v + 1u < whole; v += kShifted * kListThreads) {
        Raw<T> raw[kShifted];
#pragma unroll
        for (uint32_t b = 0; b < kShifted; ++b)
          if (v + b * kListThreads + 1u < whole)
            raw[b].template load_shifted_by<decltype(shift)::value>(
                from - d + (v + b * kListThreads) * kVecBytes<T>, (d & 2u) * 8u);
#pragma unroll
        for (uint32_t b = 0; b < kShifted; ++b)
          if (v + b * kListThreads + 1u < whole)
            clip_raw<T, O>(raw[b], f, to + (v + b * kListThreads) * kVecBytes<O>);
      }
    });
    if (whole) {
      head += kVec;
      tail = whole > 1u ? tail - kVec : head;
    }
  }
  const ClipFactor f(state.clip, scale);
  for (uint32_t e = unit_thread(); e < head + (count - tail); e += kListThreads) {
    const uint32_t i = e < head ? e : tail + (e - head);
    store1<O>(dst, i, f(from_bits<T>(elem_bits<T>(src, i))));
  }
}

// Rows on either side where every vector is one aligned run on both.
template <uint32_t T, uint32_t O, bool kSame, typename S>
__device__ __forceinline__ void clip_row_vectors(const GradUnit& u, const GradUnit& o, float scale,
                                                 S& state) {
  constexpr uint32_t kBatch = T == kGradF32 ? 2 : 4;
  if (!state.ready()) return;
  const ClipFactor f(state.clip, scale);
  uint32_t e = unit_thread() * kVec;
  Rows<T> src(u, e);
  Rows<O> dst(kSame ? u : o, e);
  for (; e < u.count; e += kBatch * kListThreads * kVec) {
    Raw<T> raw[kBatch];
    uint8_t* to[kBatch];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      if (e + b * (kListThreads * kVec) < u.count) raw[b].load(src.p, l2_first_out());
      to[b] = kSame ? src.p : dst.p;
      src.next_vector();
      if (!kSame) dst.next_vector();
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b)
      if (e + b * (kListThreads * kVec) < u.count) clip_raw<T, O>(raw[b], f, to[b]);
  }
}

// Any rows.  With rows in and contiguous memory out, vectors start at the
// output's boundaries.
template <uint32_t T, uint32_t O, typename S>
__device__ __forceinline__ void clip_rows(const GradUnit& u, const GradUnit& o, float scale,
                                          S& state) {
  if (!state.ready()) return;
  const ClipFactor f(state.clip, scale);
  const uint32_t head = o.flags & kGradPitched ? 0u : peel_of<O>(o.ptr, u.count);
  uint32_t e = head + unit_thread() * kVec;
  Rows<T> src(u, e);
  Rows<O> dst(o, e);
  for (; e < u.count; e += kListThreads * kVec) {
    const uint32_t n = vector_elems(e, u.count);
    Raw<T> raw;
    src.load(raw, n, inside_unit(u, e), l2_first_out());
    if (n == kVec && dst.aligned()) {
      clip_raw<T, O>(raw, f, dst.p);
    } else {
      float x[8];
      raw.unpack(x);
      Rows<O> to = dst;
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) {
        if (j < n) {
          store1<O>(to.p, 0, f(x[j]));
          to.next_element();
        }
      }
    }
    src.next_vector();
    dst.next_vector();
  }
  if (unit_thread() < head)
    store1<O>(Rows<O>(o, unit_thread()).p, 0,
              f(from_bits<T>(elem_bits<T>(Rows<T>(u, unit_thread()).p, 0))));
}

// kRows: kNoRows, kRowVectors, kAnyRows, each with the registers it needs.
template <uint32_t T, uint32_t O, uint32_t kRows, bool kSame, typename S>
__device__ __forceinline__ void clip_unit(const GradUnit& u, const GradUnit& o, float scale,
                                          S& state) {
  if (kRows == kRowVectors && ((u.flags | o.flags) & kGradPitched))
    clip_row_vectors<T, O, kSame>(u, o, scale, state);
  else if (kRows == kAnyRows && ((u.flags | o.flags) & kGradPitched))
    clip_rows<T, O>(u, o, scale, state);
  else
    clip_flat<T, O, kRows == kRowVectors, kRows != kRowVectors && !kSame>(
        static_cast<const uint8_t*>(u.ptr), static_cast<uint8_t*>(const_cast<void*>(o.ptr)),
        u.count, scale, state);
}

// Unit i in any layout and type on either side, element by element.  The launch
// chooses the form for vectors by the addresses that the host knows; a bind in a
// replayed graph, or one behind a captured clip, may have brought others by the
// time the kernel runs.  A call of its own, for the registers of that form's sake.
__device__ __noinline__ void clip_elements(const GradUnit* units, const GradUnit* outs, uint32_t i,
                                           float scale, float clip) {
  const GradUnit u = load_unit<true>(units, i), o = load_unit<true>(outs, i);
  const ClipFactor f(clip, scale);
  const uint32_t from = u.flags & kGradTypeMask, to = o.flags & kGradTypeMask;
#pragma unroll 1
  for (uint32_t e = unit_thread(); e < u.count; e += kListThreads) {
    const void* p = from == kGradF32 ? Rows<kGradF32>(u, e).p : Rows<kGradF16>(u, e).p;
    void* q = to == kGradF32 ? Rows<kGradF32>(o, e).p : Rows<kGradF16>(o, e).p;
    const float y = f(from == kGradF32    ? from_bits<kGradF32>(elem_bits<kGradF32>(p, 0))
                      : from == kGradBf16 ? from_bits<kGradBf16>(elem_bits<kGradBf16>(p, 0))
                                          : from_bits<kGradF16>(elem_bits<kGradF16>(p, 0)));
    if (to == kGradF32)
      store1<kGradF32>(q, 0, y);
    else if (to == kGradBf16)
      store1<kGradBf16>(q, 0, y);
    else
      store1<kGradF16>(q, 0, y);
  }
}

// kOut: the output type (units written in another one are left to the launch for
// theirs), or in place: three pairs of types a kernel, not nine, for its registers.
constexpr uint32_t kOutSame = 3u;
template <uint32_t kOut, uint32_t kRows, typename S>
__device__ __forceinline__ void clip_any(const GradListView& list, const GradListView& out,
                                         uint32_t i, float scale, S& state) {
  constexpr bool kSame = kOut == kOutSame;
  const GradUnit u = load_unit<kRows != kNoRows>(list.units, i);
  const GradUnit o = kSame ? u : load_unit<kRows != kNoRows>(out.units, i);
  if (!kSame && (o.flags & kGradTypeMask) != kOut) return;
  if (kRows == kRowVectors && !(u.flags & o.flags & kGradVector)) {
    if (state.ready())
      clip_elements(list.units, kSame ? list.units : out.units, i, scale, state.clip);
    return;
  }
  switch (u.flags & kGradTypeMask) {
    case kGradF32:
      return clip_unit<kGradF32, kSame ? kGradF32 : kOut, kRows, kSame>(u, o, scale, state);
    case kGradBf16:
      return clip_unit<kGradBf16, kSame ? kGradBf16 : kOut, kRows, kSame>(u, o, scale, state);
    default:
      return clip_unit<kGradF16, kSame ? kGradF16 : kOut, kRows, kSame>(u, o, scale, state);
  }
}

template <uint32_t kOut, uint32_t kRows, bool kOwn>
__global__ void __launch_bounds__(kListThreads,
                                  kRows == kAnyRows || (kRows && kOut == kOutSame) ? 3 : 4)
    list_clip_kernel(GradListView list, GradListView out, float scale,
                     const __grid_constant__ ClipNorm norm) {
  ClipState<kOwn> state{&norm, scale, 0.0f, 0.0f, false};
  // In place with a loss scale of one there may be nothing to do: look before
  // anything is loaded.
  if (kOut == kOutSame && scale == 1.0f && (!state.ready() || state.clip == 1.0f)) return;
  // From the end of the list to its start: the norm pass has read the end last,
  // so the part of the gradients that the L2 still holds is read first.
  if constexpr (kOut == kOutSame) {
    for (uint32_t b = blockIdx.x; b < list.n_units; b += gridDim.x)
      clip_any<kOut, kRows>(list, out, list.n_units - 1u - b, scale, state);
  } else {
    clip_any<kOut, kRows>(list, out, list.n_units - 1u - blockIdx.x, scale, state);
  }
}

// ---- small lists -------------------------------------------------------------------
// One launch of one thread-block cluster for lists whose time is latency: the
// partials, a cluster barrier, and the norm (every block for itself where it
// goes on to clip) from the same tree.  A block works on 4 units at a time; unit
// i goes to block i % cluster first.  16 blocks (8 where 16 do not fit) of 1,024
// threads: 0.1M bf16 in 9 tensors 7.6 us a call, of which 5.0 on the GPU, against
// 10.2 us for the two kernels; 8 blocks are slower from 0.25M on, 4 much.
constexpr uint32_t kSmallThreads = 1024;
constexpr uint32_t kSmallGroups = kSmallThreads / kListThreads;
constexpr uint32_t kSmallNorm = 4u, kSmallStep = 5u;  // kMode; 0..3: clip to kOut

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// The tree over at most 1,024 partials by one warp; valid in lane 0.
__device__ __forceinline__ void sum_partials_warp(const GradPartial* partials, uint32_t count,
                                                  double& sum, uint32_t& top) {
  const uint32_t lane = threadIdx.x & 31u;
  double mine = 0.0;
  top = 0u;
  for (uint32_t w = 0; w * 32u < count; ++w) {
    const uint32_t i = w * 32u + lane;
    const uint4 q = i < count ? __ldcg(reinterpret_cast<const uint4*>(partials + i))
                              : make_uint4(0u, 0u, 0u, 0u);
    const double s =
        __shfl_sync(kFull, fold_warp(__hiloint2double(int(q.y), int(q.x))), 0);
    if (lane == w) mine = s;
    top = max(top, q.z);
  }
  sum = fold_warp(mine);
  top = __reduce_max_sync(kFull, top);
}

template <uint32_t kMode>
__global__ void __launch_bounds__(kSmallThreads, 1)
    list_small_kernel(GradListView list, GradListView to, float scale, float max_norm, int kind,
                      GradListOut out, GradPartial* partials, DeviceScaler* scaler,
                      DeviceStepState* st, FinalizeParams fp) {
  __shared__ UnitSlot slots[kSmallGroups];
  __shared__ LaneSlot lanes;
  __shared__ float2 s_clip;
  constexpr bool kClip = kMode <= kOutSame;
  const uint32_t group = threadIdx.x / kListThreads;
  const uint32_t begin = blockIdx.x + gridDim.x * group, step = gridDim.x * kSmallGroups;
  pdl_wait();
  if (!kClip) pdl_trigger();  // a clip's outputs may be what the next kernel loads early
  if (kMode == kSmallStep && fp.dynamic) scale = scaler->scale;
  const float factor = square_factor(scale);
  for (uint32_t i = begin; i < list.n_units; i += step) {
    unit_partial<true>(list, load_unit<true>(list.units, i), factor, slots[group], 1u + group,
                       partials + i);
    unit_barrier(1u + group);  // the slot is free again
  }
  cluster_barrier();
  if (kClip || blockIdx.x == 0u) {
    double sum;
    uint32_t top;
    sum_partials<kSmallThreads>(partials, list.n_units, threadIdx.x, 0u, lanes, sum, top);
    if (threadIdx.x == 0u) {
      if constexpr (kMode == kSmallStep) {
        write_step(sum, top, scaler, st, fp);
      } else {
        const float4 v = norm_values(sum, top, scale, max_norm, kind);
        s_clip = make_float2(v.y, v.w);
        if (blockIdx.x == 0u) write_norm(out, v, unscaled_sum(sum, scale));
      }
    }
  }
  if (kMode != kSmallStep && (out.tensor_norms || out.tensor_max)) {
    const uint32_t warp = blockIdx.x + gridDim.x * (threadIdx.x / 32u);
    for (uint32_t t = warp; t < list.n_tensors; t += gridDim.x * (kSmallThreads / 32u)) {
      const uint32_t first = __ldg(&list.tensors[t].first_unit);
      const uint32_t end =
          t + 1u < list.n_tensors ? __ldg(&list.tensors[t + 1u].first_unit) : list.n_units;
      double sum;
      uint32_t top;
      sum_partials_warp(partials + first, end - first, sum, top);
      if ((threadIdx.x & 31u) == 0u) write_tensor(out, t, sum, top, scale, kind);
    }
  }
  if constexpr (kClip) {
    __syncthreads();
    ClipState<false> state{nullptr, scale, s_clip.x, s_clip.y, true};
    if (!state.ready() || (kMode == kOutSame && scale == 1.0f && state.clip == 1.0f)) return;
    for (uint32_t i = begin; i < list.n_units; i += step)
      clip_any<kMode, kAnyRows>(list, to, i, scale, state);
  }
}

// ---- accumulate ------------------------------------------------------------------
// acc = micro or acc + micro, one f32 rounding an element: 10 bytes an element from
// bf16 (6 to start an update), so DRAM alone bounds it.  32-byte loads and stores
// of the accumulator, everything first to leave the L2, 8,192 elements a block:
// 135M from bf16 in 201-204 us (6.7 TB/s; a plain copy reaches 6.57), 216 us with
// 2,048 a block, 204 with 16,384.
constexpr uint32_t kAccElems = 8192;
__device__ __forceinline__ void load_acc(const float* p, float (&y)[8]) {
  asm volatile("ld.global.L1::no_allocate.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]), "=f"(y[4]), "=f"(y[5]),
                 "=f"(y[6]), "=f"(y[7])
               : "l"(p)
               : "memory");
}

template <uint32_t T>
__device__ __forceinline__ void add_raw(const Raw<T>& raw, const float (&old)[8], bool overwrite,
                                        float* to) {
  float y[8];
  raw.unpack(y);
  if (!overwrite) {
#pragma unroll
    for (uint32_t j = 0; j < kVec; ++j) y[j] = __fadd_rn(old[j], y[j]);
  }
  store8<kGradF32>(to, y);
}
template <uint32_t T>
__device__ __forceinline__ void add_one(const void* src, uint64_t i, bool overwrite, float* to) {
  const float x = from_bits<T>(elem_bits<T>(src, i));
  *to = overwrite ? x : __fadd_rn(*to, x);
}

// acc[offset + e] = micro, or += micro (f32).  Vectors start at the
// accumulator's boundaries; the input is shifted where it lies off them.
template <uint32_t T>
__device__ __forceinline__ void accumulate_flat(const uint8_t* src, float* dst, uint32_t count,
                                                bool overwrite) {
  constexpr uint32_t kBatch = 2;
  const uint32_t peel = peel_of<kGradF32>(dst, count);
  const uint8_t* from = src + peel * kSize<T>;
  float* to = dst + peel;
  const uint32_t whole = (count - peel) / kVec;
  uint32_t head = peel, tail = peel + whole * kVec;  // left over: [0, head), [tail, count)
  if (reinterpret_cast<uintptr_t>(from) % kVecBytes<T> == 0u) {
    for (uint32_t v = unit_thread(); v < whole; v += kBatch * kListThreads) {
      Raw<T> raw[kBatch];
      float old[kBatch][8];
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const uint32_t i = v + b * kListThreads;
        if (i < whole) {
          raw[b].load(from + i * kVecBytes<T>, l2_first_out());
          if (!overwrite) load_acc(to + i * kVec, old[b]);
        }
      }
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const uint32_t i = v + b * kListThreads;
        if (i < whole) add_raw<T>(raw[b], old[b], overwrite, to + i * kVec);
      }
    }
  } else {
    // The blocks of the first and the last vector can reach beyond the tensor.
    for (uint32_t v = unit_thread() + 1u; v + 1u < whole; v += kListThreads) {
      Raw<T> raw;
      float old[8];
      raw.load_shifted(from + v * kVecBytes<T>);
      if (!overwrite) load_acc(to + v * kVec, old);
      add_raw<T>(raw, old, overwrite, to + v * kVec);
    }
    if (whole) {
      head += kVec;
      tail = whole > 1u ? tail - kVec : head;
    }
  }
  for (uint32_t e = unit_thread(); e < head + (count - tail); e += kListThreads) {
    const uint32_t i = e < head ? e : tail + (e - head);
    add_one<T>(src, i, overwrite, dst + i);
  }
}

template <uint32_t T>
__device__ __forceinline__ void accumulate_rows(const GradUnit& u, float* dst, bool overwrite) {
  const uint32_t count = u.count;
  const uint32_t head = peel_of<kGradF32>(dst, count);
  uint32_t e = head + unit_thread() * kVec;
  Rows<T> src(u, e);
  for (; e < count; e += kListThreads * kVec) {
    const uint32_t n = vector_elems(e, count);
    Raw<T> raw;
    float old[8];
    if (!overwrite && n == kVec) load_acc(dst + e, old);
    src.load(raw, n, inside_unit(u, e), l2_first_out());
    src.next_vector();
    if (n == kVec) {
      add_raw<T>(raw, old, overwrite, dst + e);
    } else {
      float x[8];
      raw.unpack(x);
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j)
        if (j < n) dst[e + j] = overwrite ? x[j] : __fadd_rn(dst[e + j], x[j]);
    }
  }
  if (unit_thread() < head)
    add_one<T>(Rows<T>(u, unit_thread()).p, 0, overwrite, dst + unit_thread());
}

template <uint32_t T, bool kRows>
__device__ __forceinline__ void accumulate_unit(const GradUnit& u, float* acc, bool overwrite) {
  float* dst = acc + u.offset;
  if (kRows && (u.flags & kGradPitched))
    accumulate_rows<T>(u, dst, overwrite);
  else
    accumulate_flat<T>(static_cast<const uint8_t*>(u.ptr), dst, u.count, overwrite);
}

// Elements [begin, begin + n) of a unit as a unit of their own.
template <bool kRows>
__device__ __forceinline__ void slice_unit(GradUnit& u, uint32_t begin, uint32_t n) {
  uint64_t at = begin;
  if (kRows && (u.flags & kGradPitched)) {
    const uint32_t k = u.column + begin;
    const uint32_t row = k / u.columns;
    const uint32_t column = k - row * u.columns;
    at = row * u.row_stride + column - u.column;
    u.column = column;
  }
  u.ptr = static_cast<const uint8_t*>(u.ptr) + at * elem_bytes(u.flags & kGradTypeMask);
  u.offset += begin;
  u.count = u.count - begin < n ? u.count - begin : n;
  if (begin > 0u) u.index = 1u;  // not at the tensor's start
}

// A block per kAccElems elements of a unit.
template <bool kRows>
__global__ void __launch_bounds__(kListThreads, 4)
    list_accumulate_kernel(GradListView list, uint32_t blocks_per_unit, float* acc,
                           int overwrite) {
  const uint32_t unit = blockIdx.x / blocks_per_unit;
  const uint32_t begin = (blockIdx.x - unit * blocks_per_unit) * kAccElems;
  pdl_wait();  // a bind just ahead writes the unit's record
  pdl_trigger();  // whoever starts early waits for this kernel before it reads
  GradUnit u = load_unit<kRows>(list.units, unit);
  if (begin >= u.count) return;
  slice_unit<kRows>(u, begin, kAccElems);
  switch (u.flags & kGradTypeMask) {
    case kGradF32: return accumulate_unit<kGradF32, kRows>(u, acc, overwrite != 0);
    case kGradBf16: return accumulate_unit<kGradBf16, kRows>(u, acc, overwrite != 0);
    default: return accumulate_unit<kGradF16, kRows>(u, acc, overwrite != 0);
  }
}

// The last micro-batch: accumulates the unit's vectors in the tree's order (from
// its first element, the last one padded with +0.0) and adds the squares of the
// sums.  135M bf16 in 205 us (accumulate alone 201-204); where the accumulator's vectors are
// off its 32-byte boundaries, as behind odd sizes, it is read and written value by
// value: 9M in 61 odd-sized tensors 27.9 us against 11.5.
template <uint32_t T, bool kFactor>
__device__ __forceinline__ double accumulate_squares(const GradUnit& u, float* acc, bool overwrite,
                                                     float factor, uint32_t& top) {
  constexpr uint32_t kBatch = 2;
  Rows<T> src(u, unit_thread() * kVec);
  float* dst = acc + u.offset;
  const bool wide = reinterpret_cast<uintptr_t>(dst) % 32u == 0u;
  double sum = 0.0;
  uint32_t m = 0u;
  for (uint32_t v0 = unit_thread(); v0 * kVec < u.count; v0 += kBatch * kListThreads) {
    Raw<T> raw[kBatch];
    float old[kBatch][8];
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t e = (v0 + b * kListThreads) * kVec;
      const uint32_t n = vector_elems(e, u.count);
      src.load(raw[b], n, inside_unit(u, e), l2_first_out());
      src.next_vector();
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) old[b][j] = 0.0f;
      if (!overwrite) {
        if (wide && n == kVec) {
          load_acc(dst + e, old[b]);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < kVec; ++j)
            if (j < n) old[b][j] = dst[e + j];
        }
      }
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t e = (v0 + b * kListThreads) * kVec;
      const uint32_t n = vector_elems(e, u.count);
      float y[8];
      raw[b].unpack(y);
      if (!overwrite) {
#pragma unroll
        for (uint32_t j = 0; j < kVec; ++j) y[j] = __fadd_rn(old[b][j], y[j]);
      }
      if (wide && n == kVec) {
        store8<kGradF32>(dst + e, y);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kVec; ++j)
          if (j < n) dst[e + j] = y[j];
      }
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
      sum = add_vector<kFactor>(sum, y, factor);
    }
  }
  top = m;
  return sum;
}

template <bool kFactor>
__device__ __forceinline__ double accumulate_squares_any(const GradUnit& u, float* acc,
                                                         bool overwrite, float factor,
                                                         uint32_t& top) {
  switch (u.flags & kGradTypeMask) {
    case kGradF32:
      return accumulate_squares<kGradF32, kFactor>(u, acc, overwrite, factor, top);
    case kGradBf16:
      return accumulate_squares<kGradBf16, kFactor>(u, acc, overwrite, factor, top);
    default: return accumulate_squares<kGradF16, kFactor>(u, acc, overwrite, factor, top);
  }
}

// Writes what the update reads as its gradients, so it does not trigger: the
// kernels behind it start when it has completed.
__global__ void __launch_bounds__(kListThreads)
    list_accumulate_norm_kernel(GradListView list, float* acc, int overwrite, float scale,
                                const DeviceScaler* scaler, GradPartial* partials) {
  __shared__ UnitSlot slot;
  pdl_wait();  // a bind just ahead writes the unit's record
  const GradUnit u = load_unit<true>(list.units, blockIdx.x);
  const float factor = square_factor(scaler ? scaler->scale : scale);
  uint32_t top = 0u;
  const double sum = factor == 1.0f
                   ? accumulate_squares_any<false>(u, acc, overwrite != 0, factor, top)
                   : accumulate_squares_any<true>(u, acc, overwrite != 0, factor, top);
  fold_unit(sum, top, slot, 1u, partials + blockIdx.x);
}

// ---- the step's update ---------------------------------------------------------
// AdamW with the gradients where the list has them.  A block takes 1,024
// consecutive elements of one unit (so of one tensor: one type, one decay
// weight), a thread one 8-element vector of the flat state: 32-byte loads and
// stores of master / m / v, 16 of the bf16 weights.  The state's vector
// boundaries need not be the tensor's or the gradient's: a thread whose vector is
// not whole within the tensor goes element by element, and a gradient off the
// boundaries is shifted.
//
// 28 bytes an element (bf16 gradients), bound by DRAM: all loads are in flight
// before the norm is finished (pdl_wait), 62 registers and 128 threads a block keep
// 112 KB a SM on their way, and the hardware balances the blocks.  135M elements:
// step 627-647 us, of which the update 585-605 (6.4 TB/s).  The flat step's form
// (2,048-element tiles by bulk copies into shared memory, 3 blocks a SM) took
// 667 us here; 256 / 512 threads a block 663 / 688, two vectors a thread 761.
constexpr uint32_t kUpdateBlock = 128;
constexpr uint32_t kUpdateElems = kUpdateBlock * kVec;

// 8 gradients from element e of the unit on, and one.
template <uint32_t T, bool kRows>
__device__ __forceinline__ void update_grads(const GradUnit& u, uint32_t e, float (&x)[8]) {
  Raw<T> raw;
  if (kRows && (u.flags & kGradPitched)) {
    Rows<T>(u, e).load(raw, kVec, inside_unit(u, e), l2_first_out());
  } else {
    const uint8_t* p = static_cast<const uint8_t*>(u.ptr) + e * kSize<T>;
    if (reinterpret_cast<uintptr_t>(p) % kVecBytes<T> == 0u)
      raw.load(p, l2_first_out());
    else if (e >= kVec && e + 2u * kVec <= u.count)
      raw.load_shifted(p);  // its blocks lie within the unit
    else
      gather_flat(raw, p, kVec);
  }
  raw.unpack(x);
}
template <uint32_t T, bool kRows>
__device__ __forceinline__ float update_grad(const GradUnit& u, uint32_t e) {
  if (kRows && (u.flags & kGradPitched))
    return from_bits<T>(elem_bits<T>(Rows<T>(u, e).p, 0));
  return from_bits<T>(elem_bits<T>(u.ptr, e));
}

template <bool kMul>
__device__ __forceinline__ bool update_vector(float (&g)[8], float (&th)[8], float (&m)[8],
                                              float (&v)[8], float wd, const AdamwParams& p,
                                              const ScaleInfo& sc, float clip) {
  bool bad = false;
#pragma unroll
  for (uint32_t j = 0; j < kVec; ++j) {
    const float gv = __fmul_rn(unscale<kMul>(g[j], sc), clip);
    th[j] = adamw_elem(th[j], gv, m[j], v[j], wd, p, bad);
  }
  return bad;
}

template <bool kRows>
__global__ void __launch_bounds__(kUpdateBlock, 8)
    list_update_kernel(GradListView list, uint32_t blocks_per_unit, bool backwards, float* master,
                       float* mom, float* var, uint16_t* w16, const uint8_t* decay, AdamwParams p,
                       DeviceStepState* st) {
  // From the end of a list whose end is what the L2 holds after the norm.
  const uint32_t b = backwards ? gridDim.x - 1u - blockIdx.x : blockIdx.x;
  const uint32_t unit = b / blocks_per_unit;
  const GradUnit u = load_unit<kRows>(list.units, unit);
  // The vector's first element within the unit; below zero in front of a unit
  // that starts inside a vector of the state.
  const int32_t e = int32_t((b - unit * blocks_per_unit) * kUpdateElems + threadIdx.x * kVec) -
                    int32_t(u.offset % kVec);
  const int32_t count = int32_t(u.count);
  const bool whole = e >= 0 && e + int32_t(kVec) <= count;
  const uint64_t at = u.offset + int64_t(e);
  const uint32_t type = u.flags & kGradTypeMask;
  float g[8], th[8], m[8], v[8];
  if (whole) {
    load_acc(master + at, th);
    load_acc(mom + at, m);
    load_acc(var + at, v);
    if (type == kGradF32)
      update_grads<kGradF32, kRows>(u, uint32_t(e), g);
    else if (type == kGradBf16)
      update_grads<kGradBf16, kRows>(u, uint32_t(e), g);
    else
      update_grads<kGradF16, kRows>(u, uint32_t(e), g);
  }
  const float wd = __ldg(decay + u.tensor) ? p.decay_weight : p.no_decay_weight;
  pdl_wait();  // the decision is complete and visible
  if (st->skipped || st->kernel_error) return;
  const ScaleInfo sc = decode_scale(st->loss_scale_used);
  const float clip = st->clip_apply;
  bool bad = false;
  if (whole) {
    bad = sc.mul ? update_vector<true>(g, th, m, v, wd, p, sc, clip)
                 : update_vector<false>(g, th, m, v, wd, p, sc, clip);
    store8<kGradF32>(master + at, th);
    store8<kGradF32>(mom + at, m);
    store8<kGradF32>(var + at, v);
    uint32_t w[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      w[i] = uint32_t(bf16_rne_bits(th[2 * i])) | uint32_t(bf16_rne_bits(th[2 * i + 1])) << 16;
    store_words(w16 + at, w);
  } else {
    const int32_t from = e < 0 ? 0 : e, to = e + int32_t(kVec) < count ? e + int32_t(kVec) : count;
    for (int32_t k = from; k < to; ++k) {
      const float x =
          type == kGradF32    ? update_grad<kGradF32, kRows>(u, uint32_t(k))
          : type == kGradBf16 ? update_grad<kGradBf16, kRows>(u, uint32_t(k))
                              : update_grad<kGradF16, kRows>(u, uint32_t(k));
      const uint64_t i = u.offset + uint32_t(k);
      const float gv =
          __fmul_rn(sc.mul ? unscale<true>(x, sc) : unscale<false>(x, sc), clip);
      float mk = mom[i], vk = var[i];
      const float t1 = adamw_elem(master[i], gv, mk, vk, wd, p, bad);
      master[i] = t1;
      mom[i] = mk;
      var[i] = vk;
      w16[i] = bf16_rne_bits(t1);
    }
  }
  if (bad) atomicOr(&st->result_nonfinite, 1u);
}

// ---- re-pointing -----------------------------------------------------------------
__global__ void list_bind_tensors_kernel(GradTensor* tensors, GradBind bind, uint32_t begin,
                                         uint32_t n) {
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  tensors[begin + i].ptr = bind.ptr[i];
  tensors[begin + i].flags = bind.flags[i];
}
__global__ void list_bind_units_kernel(const GradTensor* tensors, GradUnit* units,
                                       uint32_t n_units, uint32_t unit_elems, uint32_t begin,
                                       uint32_t n) {
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_units) return;
  const uint32_t k = units[i].tensor;
  if (k < begin || k - begin >= n) return;
  const GradTensor& t = tensors[k];
  uint64_t at = uint64_t(units[i].index) * unit_elems;
  if (t.flags & kGradPitched) at = at / t.columns * t.row_stride + at % t.columns;
  units[i].ptr = static_cast<const uint8_t*>(t.ptr) + at * elem_bytes(t.flags & kGradTypeMask);
  units[i].flags = t.flags;
}

// Launch chained behind the kernel ahead of it on the stream (see pdl_wait).
template <typename... Args>
cudaError_t launch_chained(void (*kernel)(Args...), uint32_t grid, uint32_t block, size_t smem,
                           cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

namespace {
template <uint32_t kMode>
cudaError_t launch_small(const GradListView& list, const GradListView& to, float scale,
                         float max_norm, int kind, const GradListOut& out, GradPartial* partials,
                         DeviceScaler* scaler, DeviceStepState* st, const FinalizeParams& fp,
                         cudaStream_t stream) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = list.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(list.cluster);
  cfg.blockDim = dim3(kSmallThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, list_small_kernel<kMode>, list, to, scale, max_norm, kind, out,
                            partials, scaler, st, fp);
}

template <uint32_t kMode>
bool small_fits(uint32_t cluster) {
  if (cluster > 8 &&
      cudaFuncSetAttribute(list_small_kernel<kMode>,
                           cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(kSmallThreads);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, list_small_kernel<kMode>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return n > 0;
}
bool all_small_fit(uint32_t c) {
  return small_fits<kGradF32>(c) && small_fits<kGradBf16>(c) && small_fits<kGradF16>(c) &&
         small_fits<kOutSame>(c) && small_fits<kSmallNorm>(c) && small_fits<kSmallStep>(c);
}

cudaError_t launch_norm_kernel(const GradListView& list, float scale, const DeviceScaler* scaler,
                               GradPartial* partials, cudaStream_t stream) {
  return launch_chained(list.rows ? list_norm_kernel<true> : list_norm_kernel<false>, list.n_units,
                        kListThreads, 0, stream, list, scale, scaler, partials);
}

// A list small enough for one cluster, on a device that can hold one.
bool is_small(const GradListView& list, uint32_t units) {
  return list.cluster != 0u && list.n_units <= units;
}
}  // namespace

uint32_t list_small_cluster() {
  // Looked up once per device (the answer, plus one).
  constexpr int kMaxDevices = 64;
  static std::atomic<uint32_t> known[kMaxDevices];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return 0u;
  uint32_t c = known[device].load(std::memory_order_acquire);
  if (c == 0u) {
    c = 1u + (all_small_fit(16u) ? 16u : all_small_fit(8u) ? 8u : 0u);
    known[device].store(c, std::memory_order_release);
  }
  return c - 1u;
}

cudaError_t launch_list_norm(const GradListView& list, float scale, float max_norm, int kind,
                             const GradListOut& out, GradPartial* partials, cudaStream_t stream) {
  if (is_small(list, kGradSmallNorm))
    return launch_small<kSmallNorm>(list, list, scale, max_norm, kind, out, partials, nullptr,
                                    nullptr, FinalizeParams{}, stream);
  if (list.n_units > 0) {
    const cudaError_t e = launch_norm_kernel(list, scale, nullptr, partials, stream);
    if (e != cudaSuccess) return e;
  }
  const uint32_t tensors = out.tensor_norms || out.tensor_max ? list.n_tensors : 0u;
  const uint32_t grid = 1u + (tensors + kTensorsPerBlock - 1u) / kTensorsPerBlock;
  return launch_chained(list_finalize_kernel, grid, kLanes, 0, stream, list,
                        static_cast<const GradPartial*>(partials), scale, max_norm, kind, out);
}

cudaError_t launch_list_norm_decide(const GradListView& list, GradPartial* partials,
                                    DeviceScaler* scaler, DeviceStepState* st,
                                    const FinalizeParams& fp, cudaStream_t stream) {
  if (is_small(list, kGradSmallStep))
    return launch_small<kSmallStep>(list, list, fp.static_scale, 1.0f, 0, GradListOut{}, partials,
                                    scaler, st, fp, stream);
  const cudaError_t e = launch_norm_kernel(list, fp.static_scale, fp.dynamic ? scaler : nullptr,
                                           partials, stream);
  if (e != cudaSuccess) return e;
  return launch_list_decide(list, partials, scaler, st, fp, stream);
}

cudaError_t launch_list_decide(const GradListView& list, const GradPartial* partials,
                               DeviceScaler* scaler, DeviceStepState* st,
                               const FinalizeParams& fp, cudaStream_t stream) {
  return launch_chained(list_decide_kernel, 1u, kLanes, 0, stream, list, partials, scaler,
                        st, fp);
}

namespace {
template <uint32_t kOut>
cudaError_t launch_clip_to(const GradListView& list, const GradListView& out, float scale,
                           const ClipNorm& norm, cudaStream_t stream) {
  const bool own = norm.result == nullptr;
  const auto kernel =
      !list.rows && !out.rows
          ? (own ? list_clip_kernel<kOut, kNoRows, true> : list_clip_kernel<kOut, kNoRows, false>)
      : list.off_runs || out.off_runs
          ? list_clip_kernel<kOut, kAnyRows, true>
          : (own ? list_clip_kernel<kOut, kRowVectors, true>
                 : list_clip_kernel<kOut, kRowVectors, false>);
  // Where there may be nothing to do, one wave of blocks that walk the units, so
  // that leaving is quick (135M below the limit: 44.7 us with the norm, against 76
  // for a block per unit); else a block per unit, which the hardware balances.
  uint32_t grid = list.n_units;
  if (kOut == kOutSame && scale == 1.0f)
    grid = std::min(grid, list.sms * (list.rows ? 3u : 4u));  // as its launch bounds
  return launch_chained(kernel, grid, kListThreads, 0, stream, list, out, scale, norm);
}
}  // namespace

cudaError_t launch_list_clip(const GradListView& list, const GradListView& to, bool in_place,
                             float scale, float max_norm, int kind, const GradListOut& out,
                             GradPartial* partials, cudaStream_t stream) {
  const bool one_type = in_place || (to.types & (to.types - 1u)) == 0u;
  if (is_small(list, kGradSmallClip) && one_type) {
    const auto launch = in_place ? launch_small<kOutSame>
                        : to.types == 1u << kGradF32  ? launch_small<kGradF32>
                        : to.types == 1u << kGradBf16 ? launch_small<kGradBf16>
                                                      : launch_small<kGradF16>;
    return launch(list, to, scale, max_norm, kind, out, partials, nullptr, nullptr,
                  FinalizeParams{}, stream);
  }
  ClipNorm norm{out.result, partials, list.n_units, max_norm, kind, out};
  cudaError_t e = cudaSuccess;
  if (one_type && list.n_units > 0u && list.n_units <= kGradOwnNorm && !out.tensor_norms &&
      !out.tensor_max) {
    norm.result = nullptr;
    e = launch_norm_kernel(list, scale, nullptr, partials, stream);
  } else {
    e = launch_list_norm(list, scale, max_norm, kind, out, partials, stream);
  }
  if (e != cudaSuccess || list.n_units == 0) return e;
  if (in_place) return launch_clip_to<kOutSame>(list, list, scale, norm, stream);
  if (to.types & (1u << kGradF32)) e = launch_clip_to<kGradF32>(list, to, scale, norm, stream);
  if (e == cudaSuccess && (to.types & (1u << kGradBf16)))
    e = launch_clip_to<kGradBf16>(list, to, scale, norm, stream);
  if (e == cudaSuccess && (to.types & (1u << kGradF16)))
    e = launch_clip_to<kGradF16>(list, to, scale, norm, stream);
  return e;
}

cudaError_t launch_list_accumulate(const GradListView& list, float* acc, int overwrite,
                                   cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  const uint32_t per_unit = list.unit_elems / kAccElems;
  const uint64_t blocks = uint64_t(list.n_units) * per_unit;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  return launch_chained(list.rows ? list_accumulate_kernel<true> : list_accumulate_kernel<false>,
                        uint32_t(blocks), kListThreads, 0, stream, list, per_unit, acc, overwrite);
}

cudaError_t launch_list_accumulate_norm(const GradListView& list, float* acc, int overwrite,
                                        float scale, const DeviceScaler* scaler,
                                        GradPartial* partials, cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  return launch_chained(list_accumulate_norm_kernel, list.n_units, kListThreads, 0, stream, list,
                        acc, overwrite, scale, scaler, partials);
}

cudaError_t launch_list_update(const GradListView& list, float* master, float* moment,
                               float* variance, uint16_t* w16, const uint8_t* decay,
                               const AdamwParams& p, DeviceStepState* st, bool chained,
                               cudaStream_t stream) {
  // One block more where a unit can start inside a vector of the state.
  const uint32_t per_unit = list.unit_elems / kUpdateElems + (list.off_vectors ? 1u : 0u);
  const uint64_t blocks = uint64_t(list.n_units) * per_unit;
  if (blocks == 0 || blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  const auto kernel = list.rows ? list_update_kernel<true> : list_update_kernel<false>;
  if (chained)
    return launch_chained(kernel, uint32_t(blocks), kUpdateBlock, 0, stream, list, per_unit,
                          list.keep > 0u, master, moment, variance, w16, decay, p, st);
  kernel<<<uint32_t(blocks), kUpdateBlock, 0, stream>>>(list, per_unit, list.keep > 0u, master,
                                                        moment, variance, w16, decay, p, st);
  return cudaGetLastError();
}

cudaError_t launch_list_bind(GradTensor* tensors, GradUnit* units, uint32_t n_units,
                             uint32_t unit_elems, const GradBind& bind, uint32_t begin, uint32_t n,
                             cudaStream_t stream) {
  list_bind_tensors_kernel<<<1, kGradBindBatch, 0, stream>>>(tensors, bind, begin, n);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || n_units == 0) return e;
  list_bind_units_kernel<<<(n_units + 255) / 256, 256, 0, stream>>>(tensors, units, n_units,
                                                                    unit_elems, begin, n);
  return cudaGetLastError();
}

}  // namespace slmopt
