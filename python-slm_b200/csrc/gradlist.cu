// Kernels over gradient lists: tensors that lie where the backward pass left
// them, in f32, bf16 or f16, contiguous or as rows with a pitch.
//
//   list_norm_kernel        -- one block per unit: unscale, squares, the unit's
//                              f64 partial and largest magnitude.
//   list_finalize_kernel    -- block 0: norm, clip scale, non-finite flag; one
//                              more block per tensor for the tensors' own norms.
//   list_clip_kernel        -- one block per unit: unscale, clip, write.
//   list_accumulate_kernel  -- one block per unit: into the flat f32 accumulator
//                              (and the partials of the sums, last micro-batch).
//   list_decide_kernel, list_update_kernel -- the optimizer step on a list.
//
// All of them stream; nothing is a contraction.  The kernels of one call are
// chained by programmatic dependent launch: each lets the next one become
// resident at once and the next one waits for its results (pdl_wait) after it
// has issued what loads do not depend on them.
#include "step_device.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace slmopt {
namespace {

constexpr uint32_t kListThreads = 256;
constexpr uint32_t kFinalThreads = 512;

// ---- element types ------------------------------------------------------------
// Raw<T>: 8 elements as they lie in memory, kept packed while loads are in flight.
template <uint32_t T>
struct Raw {
  uint4 r;
  __device__ __forceinline__ void zero() { r = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const void* p) {
    r = __ldcg(static_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    if constexpr (T == kGradBf16) {
      unpack_bf16x8(r, x);
    } else {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
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
  // Largest magnitude so far, two 16-bit lanes: without their sign, finite
  // values, infinity and NaN order as integers.
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = __vmaxu2(m, r.x & 0x7fff7fffu);
    m = __vmaxu2(m, r.y & 0x7fff7fffu);
    m = __vmaxu2(m, r.z & 0x7fff7fffu);
    m = __vmaxu2(m, r.w & 0x7fff7fffu);
  }
};
template <>
struct Raw<kGradF32> {
  uint4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const void* p) {
    a = __ldcg(static_cast<const uint4*>(p));
    b = __ldcg(static_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y);
    x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y);
    x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  }
  __device__ __forceinline__ void top(uint32_t& m) const {
    m = max(m, max(max(a.x & 0x7fffffffu, a.y & 0x7fffffffu),
                   max(a.z & 0x7fffffffu, a.w & 0x7fffffffu)));
    m = max(m, max(max(b.x & 0x7fffffffu, b.y & 0x7fffffffu),
                   max(b.z & 0x7fffffffu, b.w & 0x7fffffffu)));
  }
};

__device__ __forceinline__ uint32_t elem_bytes(uint32_t type) { return type == kGradF32 ? 4u : 2u; }

// Bits of |x| for element i, in the form Raw<T>::top keeps (16-bit types: the low lane).
template <uint32_t T>
__device__ __forceinline__ uint32_t elem_bits(const void* p, uint64_t i) {
  if constexpr (T == kGradF32)
    return static_cast<const uint32_t*>(p)[i];
  else
    return static_cast<const uint16_t*>(p)[i];
}
template <uint32_t T>
__device__ __forceinline__ float from_bits(uint32_t b) {
  if constexpr (T == kGradF32)
    return __uint_as_float(b);
  else if constexpr (T == kGradBf16)
    return __uint_as_float(b << 16);
  else
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
}

// A thread's two 16-bit lanes (or one f32) of largest magnitude, as f32 bits.
template <uint32_t T>
__device__ __forceinline__ uint32_t top_f32(uint32_t m) {
  if constexpr (T == kGradF32) {
    return m;
  } else {
    const uint32_t h = max(m & 0xffffu, m >> 16);
    return __float_as_uint(from_bits<T>(h)) & 0x7fffffffu;
  }
}

template <uint32_t T>
constexpr uint32_t kSize = T == kGradF32 ? 4u : 2u;

// Where a unit's elements lie.  `at(e)` is the address of element e of the unit
// counted in row-major order; for a vector-aligned tensor, e a multiple of 8,
// all 8 elements are one run.
template <uint32_t T>
struct Place {
  const uint8_t* base;
  uint64_t first;  // pitched: the unit's first element within its tensor
  uint64_t columns, stride;
  bool pitched;
  __device__ __forceinline__ Place(const GradUnit& u, const GradTensor* tensors,
                                   uint32_t unit_elems)
      : base(static_cast<const uint8_t*>(u.ptr)), first(0), columns(1), stride(0),
        pitched((u.flags & kGradPitched) != 0u) {
    if (pitched) {
      const GradTensor* t = tensors + u.tensor;
      columns = __ldg(&t->columns);
      stride = __ldg(&t->row_stride);
      first = uint64_t(u.index) * unit_elems;
    }
  }
  __device__ __forceinline__ uint64_t element(uint32_t e) const {
    if (!pitched) return e;
    const uint64_t k = first + e;
    uint64_t row;
    if ((k | columns) <= 0xffffffffull)
      row = static_cast<uint32_t>(k) / static_cast<uint32_t>(columns);
    else
      row = k / columns;
    return row * stride + (k - row * columns);
  }
  __device__ __forceinline__ const void* at(uint32_t e) const {
    return base + element(e) * kSize<T>;
  }
};

__device__ __forceinline__ GradUnit load_unit(const GradUnit* units, uint32_t i) {
  GradUnit u;
  const uint4* p = reinterpret_cast<const uint4*>(units + i);
  *reinterpret_cast<uint4*>(&u) = __ldg(p);
  *(reinterpret_cast<uint4*>(&u) + 1) = __ldg(p + 1);
  return u;
}

// ---- norm ----------------------------------------------------------------------
// The fixed tree of one unit: thread t owns the unit's 8-element vectors t,
// t + 256, ...; a vector's unscaled squares are added pairwise in f32
// (add_squares8) and the sums in order to the thread's f64 accumulator; elements
// past the end count as +0.0.  The block folds as the flat norm's does.
template <uint32_t T, bool kMul>
__device__ __forceinline__ double unit_squares(const GradUnit& u, const GradTensor* tensors,
                                               uint32_t unit_elems, const ScaleInfo& sc,
                                               uint32_t& top) {
  constexpr uint32_t kBatch = T == kGradF32 ? 4 : 8;  // 128 bytes of loads in flight per thread
  const Place<T> place(u, tensors, unit_elems);
  const uint32_t whole = u.count / kVec;
  double acc = 0.0;
  uint32_t m = 0u;
  if (u.flags & kGradVector) {
    for (uint32_t v0 = threadIdx.x; v0 < whole; v0 += kBatch * kListThreads) {
      Raw<T> raw[kBatch];
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const uint32_t v = v0 + b * kListThreads;
        if (v < whole)
          raw[b].load(place.at(v * kVec));
        else
          raw[b].zero();
      }
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        float x[8];
        raw[b].unpack(x);
        raw[b].top(m);
        acc = add_squares8<kMul>(acc, x, sc);
      }
    }
  } else {
    for (uint32_t v = threadIdx.x; v < whole; v += kListThreads) {
      float x[8];
      uint32_t bits[8];
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j)
        bits[j] = elem_bits<T>(place.base, place.element(v * kVec + j));
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) {
        x[j] = from_bits<T>(bits[j]);
        m = max(m, bits[j] & (T == kGradF32 ? 0x7fffffffu : 0x7fffu));
      }
      acc = add_squares8<kMul>(acc, x, sc);
    }
  }
  // The last, partial vector.
  const uint32_t rest = u.count - whole * kVec;
  if (rest && threadIdx.x == whole % kListThreads) {
    float x[8];
#pragma unroll
    for (uint32_t j = 0; j < kVec; ++j) {
      const uint32_t bits =
          j < rest ? elem_bits<T>(place.base, place.element(whole * kVec + j)) : 0u;
      x[j] = from_bits<T>(bits);
      if constexpr (T == kGradF32)
        m = max(m, bits & 0x7fffffffu);
      else
        m = __vmaxu2(m, bits & 0x7fffu);
    }
    acc = add_squares8<kMul>(acc, x, sc);
  }
  top = top_f32<T>(m);
  return acc;
}

// Folds (sum, top) over the block; results valid in thread 0.
template <uint32_t kThreads>
__device__ __forceinline__ void fold_block(double& v, uint32_t& top, double* s_sum,
                                           uint32_t* s_top) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = __dadd_rn(v, __shfl_down_sync(kFull, v, off));
  top = __reduce_max_sync(kFull, top);
  if ((threadIdx.x & 31u) == 0u) {
    s_sum[threadIdx.x >> 5] = v;
    s_top[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    constexpr int kWarps = int(kThreads / 32);
    double w[kWarps];
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      w[i] = s_sum[i];
      top = max(top, s_top[i]);
    }
#pragma unroll
    for (int off = kWarps / 2; off >= 1; off >>= 1) {
#pragma unroll
      for (int i = 0; i < off; ++i) w[i] = __dadd_rn(w[i], w[i + off]);
    }
    v = w[0];
  }
}

template <bool kMul>
__device__ __forceinline__ double unit_squares_any(const GradUnit& u, const GradTensor* tensors,
                                                   uint32_t unit_elems, const ScaleInfo& sc,
                                                   uint32_t& top) {
  switch (u.flags & kGradTypeMask) {
    case kGradF32: return unit_squares<kGradF32, kMul>(u, tensors, unit_elems, sc, top);
    case kGradBf16: return unit_squares<kGradBf16, kMul>(u, tensors, unit_elems, sc, top);
    default: return unit_squares<kGradF16, kMul>(u, tensors, unit_elems, sc, top);
  }
}

__global__ void __launch_bounds__(kListThreads)
    list_norm_kernel(GradListView list, float scale, const DeviceScaler* scaler,
                     GradPartials part) {
  __shared__ double s_sum[kListThreads / 32];
  __shared__ uint32_t s_top[kListThreads / 32];
  pdl_trigger();
  const GradUnit u = load_unit(list.units, blockIdx.x);
  const ScaleInfo sc = decode_scale(scaler ? scaler->scale : scale);
  uint32_t top = 0u;
  double sum = sc.mul ? unit_squares_any<true>(u, list.tensors, list.unit_elems, sc, top)
                      : unit_squares_any<false>(u, list.tensors, list.unit_elems, sc, top);
  fold_block<kListThreads>(sum, top, s_sum, s_top);
  if (threadIdx.x == 0) {
    part.sums[blockIdx.x] = sum;
    part.tops[blockIdx.x] = top;
  }
}

// Thread t adds partials begin + t, begin + t + 512, ... in order, 8 loads in
// flight; then the block folds.  Valid in thread 0.
__device__ __forceinline__ void sum_partials(const GradPartials& part, uint32_t begin,
                                             uint32_t count, double& v, uint32_t& top,
                                             double* s_sum, uint32_t* s_top) {
  v = 0.0;
  top = 0u;
  for (uint32_t i0 = threadIdx.x; i0 < count; i0 += 8 * kFinalThreads) {
    double q[8];
    uint32_t w[8];
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b) {
      const uint32_t i = i0 + b * kFinalThreads;
      q[b] = i < count ? __ldcg(part.sums + begin + i) : 0.0;
      w[b] = i < count ? __ldcg(part.tops + begin + i) : 0u;
    }
#pragma unroll
    for (uint32_t b = 0; b < 8; ++b) {
      v = __dadd_rn(v, q[b]);
      top = max(top, w[b]);
    }
  }
  fold_block<kFinalThreads>(v, top, s_sum, s_top);
}

__device__ __forceinline__ float unscaled_top(uint32_t top, float scale) {
  const ScaleInfo sc = decode_scale(scale);
  const float x = __uint_as_float(top);
  return sc.mul ? unscale<true>(x, sc) : unscale<false>(x, sc);
}

__global__ void __launch_bounds__(kFinalThreads)
    list_finalize_kernel(GradListView list, GradPartials part, float scale, float max_norm,
                         int kind, GradListOut out) {
  __shared__ double s_sum[kFinalThreads / 32];
  __shared__ uint32_t s_top[kFinalThreads / 32];
  pdl_trigger();
  uint32_t begin = 0u, count = list.n_units;
  if (blockIdx.x > 0) {
    const uint32_t t = blockIdx.x - 1u;
    begin = __ldg(&list.tensors[t].first_unit);
    const uint32_t end =
        t + 1u < list.n_tensors ? __ldg(&list.tensors[t + 1u].first_unit) : list.n_units;
    count = end - begin;
  }
  pdl_wait();
  double sum;
  uint32_t top;
  sum_partials(part, begin, count, sum, top, s_sum, s_top);
  if (threadIdx.x != 0) return;
  const float largest = unscaled_top(top, scale);
  const float norm = kind != 0 ? largest : __double2float_rn(__dsqrt_rn(sum));
  if (blockIdx.x > 0) {
    if (out.tensor_norms) out.tensor_norms[blockIdx.x - 1u] = norm;
    if (out.tensor_max) out.tensor_max[blockIdx.x - 1u] = largest;
    return;
  }
  const bool bad = !finite_f32(norm) || !finite_f32(largest);
  // The flat step's formula: the sum rounded once to f32, f32 root and quotient.
  const float root = kind != 0 ? largest : __fsqrt_rn(__double2float_rn(sum));
  float clip = 1.0f;
  if (bad || !finite_f32(root))
    clip = 0.0f;
  else if (root > 0.0f)
    clip = fminf(__fdiv_rn(max_norm, root), 1.0f);
  out.result[0] = norm;
  out.result[1] = clip;
  out.result[2] = largest;
  out.result[3] = bad || !finite_f32(root) ? 1.0f : 0.0f;
  if (out.sum_squares) *out.sum_squares = sum;
}

__global__ void __launch_bounds__(kFinalThreads)
    list_decide_kernel(GradListView list, GradPartials part, DeviceScaler* scaler,
                       DeviceStepState* st, FinalizeParams fp) {
  __shared__ double s_sum[kFinalThreads / 32];
  __shared__ uint32_t s_top[kFinalThreads / 32];
  pdl_trigger();
  pdl_wait();
  double sum;
  uint32_t top;
  sum_partials(part, 0u, list.n_units, sum, top, s_sum, s_top);
  if (threadIdx.x != 0) return;
  const float scale = fp.dynamic ? scaler->scale : fp.static_scale;
  const uint32_t nonfinite =
      !isfinite(sum) || !finite_f32(unscaled_top(top, scale)) ? 1u : 0u;
  const StepDecision d =
      decide_step(sum, nonfinite, scale, fp.dynamic ? scaler->good_steps : 0u, fp);
  write_decision(d, sum, nonfinite, scale, st, scaler, fp);
  st->result_nonfinite = 0u;
}

// ---- clip ----------------------------------------------------------------------
template <uint32_t T>
__device__ __forceinline__ void store8(void* p, const float (&y)[8]) {
  if constexpr (T == kGradF32) {
    __stcs(static_cast<float4*>(p), make_float4(y[0], y[1], y[2], y[3]));
    __stcs(static_cast<float4*>(p) + 1, make_float4(y[4], y[5], y[6], y[7]));
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
    __stcs(static_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}
template <uint32_t T>
__device__ __forceinline__ void store1(void* p, float y) {
  if constexpr (T == kGradF32)
    *static_cast<float*>(p) = y;
  else if constexpr (T == kGradBf16)
    *static_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(y);
  else
    *static_cast<__half*>(p) = __float2half_rn(y);
}

__device__ __forceinline__ float clipped(float x, const ScaleInfo& sc, float clip) {
  return __fmul_rn(sc.mul ? unscale<true>(x, sc) : unscale<false>(x, sc), clip);
}

// Reads and writes element by element of the same index; in place each element
// is written by the thread that read it.
template <uint32_t T, uint32_t O>
__device__ __forceinline__ void clip_unit(const GradUnit& u, const GradUnit& o,
                                          const GradListView& list, const GradListView& out,
                                          const ScaleInfo& sc, const float* result,
                                          bool in_place) {
  constexpr uint32_t kBatch = T == kGradF32 ? 4 : 8;
  const Place<T> src(u, list.tensors, list.unit_elems);
  const Place<O> dst(o, out.tensors, out.unit_elems);
  const uint32_t whole = (u.flags & o.flags & kGradVector) ? u.count / kVec : 0u;
  Raw<T> raw[kBatch];
  bool waited = false;
  float clip = 0.0f;
  for (uint32_t v0 = threadIdx.x; v0 < whole || !waited; v0 += kBatch * kListThreads) {
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t v = v0 + b * kListThreads;
      if (v < whole) raw[b].load(src.at(v * kVec));
    }
    if (!waited) {
      // The first loads are on their way; nothing is written before the clip
      // scale is there.
      pdl_wait();
      waited = true;
      clip = __ldcg(result + 1);
      const bool bad = __ldcg(result + 3) != 0.0f;
      // A non-finite gradient leaves the outputs alone; so does a product with
      // one and one in place, which changes no bit.
      if (bad || (in_place && clip == 1.0f && sc.s == 1.0f)) return;
    }
#pragma unroll
    for (uint32_t b = 0; b < kBatch; ++b) {
      const uint32_t v = v0 + b * kListThreads;
      if (v < whole) {
        float x[8];
        raw[b].unpack(x);
#pragma unroll
        for (uint32_t j = 0; j < kVec; ++j) x[j] = clipped(x[j], sc, clip);
        store8<O>(const_cast<void*>(dst.at(v * kVec)), x);
      }
    }
  }
  for (uint32_t e = whole * kVec + threadIdx.x; e < u.count; e += kListThreads) {
    const float x = from_bits<T>(elem_bits<T>(src.base, src.element(e)));
    store1<O>(const_cast<void*>(dst.at(e)), clipped(x, sc, clip));
  }
}

template <uint32_t T>
__device__ __forceinline__ void clip_unit_to(const GradUnit& u, const GradUnit& o,
                                             const GradListView& list, const GradListView& out,
                                             const ScaleInfo& sc, const float* result,
                                             bool in_place) {
  switch (o.flags & kGradTypeMask) {
    case kGradF32: return clip_unit<T, kGradF32>(u, o, list, out, sc, result, in_place);
    case kGradBf16: return clip_unit<T, kGradBf16>(u, o, list, out, sc, result, in_place);
    default: return clip_unit<T, kGradF16>(u, o, list, out, sc, result, in_place);
  }
}

__global__ void __launch_bounds__(kListThreads)
    list_clip_kernel(GradListView list, GradListView out, float scale, const float* result,
                     bool in_place) {
  // From the end of the list to its start: the norm pass has read the end last,
  // so the part of the gradients that the L2 still holds is read first.
  const uint32_t i = gridDim.x - 1u - blockIdx.x;
  const GradUnit u = load_unit(list.units, i);
  const GradUnit o = load_unit(out.units, i);
  const ScaleInfo sc = decode_scale(scale);
  switch (u.flags & kGradTypeMask) {
    case kGradF32: return clip_unit_to<kGradF32>(u, o, list, out, sc, result, in_place);
    case kGradBf16: return clip_unit_to<kGradBf16>(u, o, list, out, sc, result, in_place);
    default: return clip_unit_to<kGradF16>(u, o, list, out, sc, result, in_place);
  }
}

// ---- accumulate ------------------------------------------------------------------
// acc[offset + e] = micro, or += micro (f32), and with kNorm the unit's partial of
// the sums, in the tree of unit_squares over f32 values.
template <uint32_t T, bool kNorm, bool kMul>
__device__ __forceinline__ double accumulate_unit(const GradUnit& u, const GradListView& list,
                                                  float* acc, bool overwrite,
                                                  const ScaleInfo& sc, uint32_t& top) {
  constexpr uint32_t kBatch = T == kGradF32 ? 2 : 4;
  const Place<T> src(u, list.tensors, list.unit_elems);
  float* dst = acc + u.offset;
  const bool vector = (u.flags & kGradVector) && u.offset % 4u == 0u;
  const uint32_t whole = u.count / kVec;
  double sum = 0.0;
  uint32_t m = 0u;
  auto take = [&](const float (&y)[8]) {
    if constexpr (kNorm) {
      float x[8];
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) {
        x[j] = y[j];
        m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
      }
      sum = add_squares8<kMul>(sum, x, sc);
    }
  };
  uint32_t done = 0u;  // whole vectors done
  if (vector) {
    done = whole;
    for (uint32_t v0 = threadIdx.x; v0 < whole; v0 += kBatch * kListThreads) {
      Raw<T> raw[kBatch];
      float4 old[kBatch][2];
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const uint32_t v = v0 + b * kListThreads;
        if (v < whole) {
          raw[b].load(src.at(v * kVec));
          if (!overwrite) {
            old[b][0] = __ldcs(reinterpret_cast<const float4*>(dst + v * kVec));
            old[b][1] = __ldcs(reinterpret_cast<const float4*>(dst + v * kVec) + 1);
          }
        }
      }
#pragma unroll
      for (uint32_t b = 0; b < kBatch; ++b) {
        const uint32_t v = v0 + b * kListThreads;
        if (v < whole) {
          float y[8];
          raw[b].unpack(y);
          if (!overwrite) {
            y[0] = __fadd_rn(old[b][0].x, y[0]); y[1] = __fadd_rn(old[b][0].y, y[1]);
            y[2] = __fadd_rn(old[b][0].z, y[2]); y[3] = __fadd_rn(old[b][0].w, y[3]);
            y[4] = __fadd_rn(old[b][1].x, y[4]); y[5] = __fadd_rn(old[b][1].y, y[5]);
            y[6] = __fadd_rn(old[b][1].z, y[6]); y[7] = __fadd_rn(old[b][1].w, y[7]);
          }
          store8<kGradF32>(dst + v * kVec, y);
          take(y);
        }
      }
    }
  }
  if constexpr (kNorm) {
    // Vector by vector, in the tree's order, the last one padded with +0.0.
    for (uint32_t v = done + (threadIdx.x + kListThreads - done % kListThreads) % kListThreads;
         v * kVec < u.count; v += kListThreads) {
      float y[8];
#pragma unroll
      for (uint32_t j = 0; j < kVec; ++j) {
        const uint32_t e = v * kVec + j;
        y[j] = 0.0f;
        if (e < u.count) {
          const float x = from_bits<T>(elem_bits<T>(src.base, src.element(e)));
          y[j] = overwrite ? x : __fadd_rn(dst[e], x);
          dst[e] = y[j];
        }
      }
      take(y);
    }
    top = m;
  } else {
    for (uint32_t e = done * kVec + threadIdx.x; e < u.count; e += kListThreads) {
      const float x = from_bits<T>(elem_bits<T>(src.base, src.element(e)));
      dst[e] = overwrite ? x : __fadd_rn(dst[e], x);
    }
  }
  return sum;
}

template <bool kNorm, bool kMul>
__device__ __forceinline__ double accumulate_any(const GradUnit& u, const GradListView& list,
                                                 float* acc, bool overwrite, const ScaleInfo& sc,
                                                 uint32_t& top) {
  switch (u.flags & kGradTypeMask) {
    case kGradF32:
      return accumulate_unit<kGradF32, kNorm, kMul>(u, list, acc, overwrite, sc, top);
    case kGradBf16:
      return accumulate_unit<kGradBf16, kNorm, kMul>(u, list, acc, overwrite, sc, top);
    default:
      return accumulate_unit<kGradF16, kNorm, kMul>(u, list, acc, overwrite, sc, top);
  }
}

__global__ void __launch_bounds__(kListThreads)
    list_accumulate_kernel(GradListView list, float* acc, int overwrite) {
  const GradUnit u = load_unit(list.units, blockIdx.x);
  const ScaleInfo none{1.0f, 1.0f, true};
  uint32_t top = 0u;
  accumulate_any<false, true>(u, list, acc, overwrite != 0, none, top);
}

// Writes what the update reads as its gradients, so it does not trigger: the
// kernels behind it start when it has completed.
__global__ void __launch_bounds__(kListThreads)
    list_accumulate_norm_kernel(GradListView list, float* acc, int overwrite, float scale,
                                const DeviceScaler* scaler, GradPartials part) {
  __shared__ double s_sum[kListThreads / 32];
  __shared__ uint32_t s_top[kListThreads / 32];
  const GradUnit u = load_unit(list.units, blockIdx.x);
  const ScaleInfo sc = decode_scale(scaler ? scaler->scale : scale);
  uint32_t top = 0u;
  double sum = sc.mul ? accumulate_any<true, true>(u, list, acc, overwrite != 0, sc, top)
                      : accumulate_any<true, false>(u, list, acc, overwrite != 0, sc, top);
  fold_block<kListThreads>(sum, top, s_sum, s_top);
  if (threadIdx.x == 0) {
    part.sums[blockIdx.x] = sum;
    part.tops[blockIdx.x] = top;
  }
}

// ---- the step's update ---------------------------------------------------------
// adamw_update_bulk_kernel with its gradients fetched from the list: the state is
// walked in the flat 2,048-element tiles of that kernel (their addresses are
// always aligned), a producer warp streams master / m / v and, where the tile
// lies inside one contiguous tensor, the gradient (from the 16-byte boundary
// below its first element, if the tensor's own bytes cover that) into a
// shared-memory stage.  Tiles that mix tensors or whose tensor has a pitch read
// their gradients from global memory.
struct TileInfo {
  const uint8_t* ptr;  // the tile's tensor (staged: unused)
  uint32_t tensor;     // of the tile's first element
  uint32_t flags;      // of that tensor
  uint32_t shift;      // staged: bytes from the stage's start to the first element
  uint32_t mode;
};
constexpr uint32_t kTileStaged = 0u;  // the stage holds the gradients
constexpr uint32_t kTileOne = 1u;     // one tensor, read from global memory
constexpr uint32_t kTileMany = 2u;    // several tensors
constexpr uint32_t kListGradBytes = kBulkTile * 4 + 16;
constexpr uint32_t kListStateBytes = kBulkTile * 4;
constexpr uint32_t kListStageBytes = kListGradBytes + 3 * kListStateBytes;
static_assert(kListStageBytes % 16 == 0, "stages stay 16-byte aligned");
constexpr size_t list_update_smem() {
  return size_t(kBulkStages) * (kListStageBytes + sizeof(TileInfo)) + 128;
}

__device__ __forceinline__ float grad_value(const uint8_t* p, uint32_t type, uint64_t i) {
  switch (type) {
    case kGradF32: return from_bits<kGradF32>(elem_bits<kGradF32>(p, i));
    case kGradBf16: return from_bits<kGradBf16>(elem_bits<kGradBf16>(p, i));
    default: return from_bits<kGradF16>(elem_bits<kGradF16>(p, i));
  }
}

// Element e of the flat state within tensor k's memory (pitched or not).
__device__ __forceinline__ float grad_at(const GradTensor* tensors, uint32_t k, uint64_t local) {
  const GradTensor* t = tensors + k;
  const uint32_t flags = __ldg(&t->flags);
  uint64_t i = local;
  if (flags & kGradPitched) {
    const uint64_t columns = __ldg(&t->columns);
    const uint64_t row = (local | columns) <= 0xffffffffull
                             ? uint64_t(uint32_t(local) / uint32_t(columns))
                             : local / columns;
    i = row * __ldg(&t->row_stride) + (local - row * columns);
  }
  const uint8_t* p = reinterpret_cast<const uint8_t*>(
      __ldg(reinterpret_cast<const unsigned long long*>(&t->ptr)));
  return grad_value(p, flags & kGradTypeMask, i);
}

// 4 staged gradients from byte address p of shared memory (element-aligned).
__device__ __forceinline__ void staged4(const uint8_t* p, uint32_t type, float (&x)[4]) {
  if (type == kGradF32) {
    if ((smem_u32(p) & 15u) == 0u) {
      lds4(reinterpret_cast<const float*>(p), x);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) x[j] = reinterpret_cast<const float*>(p)[j];
    }
    return;
  }
  uint32_t h[4];
  if ((smem_u32(p) & 7u) == 0u) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    h[0] = r.x & 0xffffu; h[1] = r.x >> 16;
    h[2] = r.y & 0xffffu; h[3] = r.y >> 16;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) h[j] = reinterpret_cast<const uint16_t*>(p)[j];
  }
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    x[j] = type == kGradBf16 ? from_bits<kGradBf16>(h[j]) : from_bits<kGradF16>(h[j]);
}

// The tensor of flat element e: scanning forward from k (a tile's first tensor),
// or searching [k, n) where a tile may hold many tensors.
__device__ __forceinline__ uint32_t tensor_of(uint64_t e, uint32_t k, const uint64_t* offsets) {
  while (e >= __ldg(offsets + k + 1)) ++k;
  return k;
}
__device__ __forceinline__ uint32_t search_tensor(uint64_t e, uint32_t k, uint32_t n,
                                                  const uint64_t* offsets) {
  uint32_t hi = n;  // offsets[k] <= e < offsets[hi]
  while (hi - k > 1u) {
    const uint32_t mid = k + (hi - k) / 2u;
    if (e >= __ldg(offsets + mid))
      k = mid;
    else
      hi = mid;
  }
  return k;
}

template <bool kMul>
__device__ __forceinline__ bool list_consume(uint8_t* smem, const TileInfo* infos,
                                             uint64_t* full_bar, uint64_t* empty_bar,
                                             uint64_t n_full, const GradListView& list,
                                             float* __restrict__ master, float* __restrict__ mom,
                                             float* __restrict__ var, uint16_t* __restrict__ w16,
                                             const uint64_t* __restrict__ offsets,
                                             const uint8_t* __restrict__ decay,
                                             const AdamwParams& p, const ScaleInfo& sc,
                                             float clip, bool& bad) {
  const uint32_t t = threadIdx.x;
  uint32_t i = 0;
  for (uint64_t tile = blockIdx.x; tile < n_full; tile += gridDim.x, ++i) {
    const uint32_t s = i % kBulkStages;
    if (!mbar_wait(&full_bar[s], (i / kBulkStages) & 1u)) return false;
    const TileInfo info = infos[s];
    const uint64_t tile0 = tile * kBulkTile;
    const uint8_t* base = smem + size_t(s) * kListStageBytes;
    const float* sm = reinterpret_cast<const float*>(base + kListGradBytes);
    const float* s1 = sm + kBulkTile;
    const float* s2 = s1 + kBulkTile;
    const uint32_t type = info.flags & kGradTypeMask;
    const float wd_tile = __ldg(decay + info.tensor) ? p.decay_weight : p.no_decay_weight;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t o = h * (kBulkTile / 2) + 4 * t;
      const uint64_t e0 = tile0 + o;
      float gx[4], th[4], mm[4], vv[4], wd[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) wd[j] = wd_tile;
      if (info.mode == kTileStaged) {
        staged4(base + info.shift + o * elem_bytes(type), type, gx);
      } else {
        uint32_t k = info.tensor;
        if (info.mode == kTileMany) k = search_tensor(e0, k, list.n_tensors, offsets);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          if (info.mode == kTileMany) {
            k = tensor_of(e0 + j, k, offsets);
            wd[j] = __ldg(decay + k) ? p.decay_weight : p.no_decay_weight;
          }
          gx[j] = grad_at(list.tensors, k, e0 + j - __ldg(offsets + k));
        }
      }
      lds4(sm + o, th);
      lds4(s1 + o, mm);
      lds4(s2 + o, vv);
      uint32_t bits[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const float gv = __fmul_rn(unscale<kMul>(gx[j], sc), clip);
        th[j] = adamw_elem(th[j], gv, mm[j], vv[j], wd[j], p, bad);
        bits[j] = bf16_rne_bits(th[j]);
      }
      __stcs(reinterpret_cast<float4*>(master + e0), make_float4(th[0], th[1], th[2], th[3]));
      __stcs(reinterpret_cast<float4*>(mom + e0), make_float4(mm[0], mm[1], mm[2], mm[3]));
      __stcs(reinterpret_cast<float4*>(var + e0), make_float4(vv[0], vv[1], vv[2], vv[3]));
      __stcs(reinterpret_cast<uint2*>(w16 + e0),
             make_uint2(bits[0] | (bits[1] << 16), bits[2] | (bits[3] << 16)));
    }
    __syncwarp();
    if ((t & 31) == 0) mbar_arrive(&empty_bar[s]);
  }
  return true;
}

__global__ void __launch_bounds__(kBulkThreads)
    list_update_kernel(GradListView list, float* __restrict__ master, float* __restrict__ mom,
                       float* __restrict__ var, uint16_t* __restrict__ w16,
                       const uint64_t* __restrict__ offsets, const uint8_t* __restrict__ decay,
                       const uint32_t* __restrict__ tile_first, AdamwParams p,
                       DeviceStepState* st) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_scale, s_clip;
  __shared__ uint32_t s_go, s_stop;
  TileInfo* infos = reinterpret_cast<TileInfo*>(smem + size_t(kBulkStages) * kListStageBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(infos + kBulkStages);
  uint64_t* empty_bar = full_bar + kBulkStages;
  const uint64_t n = list.elements;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kBulkStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], kBulkConsumers / 32);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_stop = 0u;
  }
  __syncthreads();
  const uint64_t n_full = n / kBulkTile;
  const uint64_t mine = n_full > blockIdx.x ? (n_full - 1u - blockIdx.x) / gridDim.x + 1u : 0u;
  bool ok = true;
  bool bad = false;
  uint32_t i = 0;  // producer: tiles issued
  if (threadIdx.x >= kBulkConsumers) {
    if (threadIdx.x == kBulkConsumers) {
      for (uint64_t tile = blockIdx.x; tile < n_full; tile += gridDim.x, ++i) {
        const uint32_t s = i % kBulkStages;
        if (i >= kBulkStages) {
          if (!mbar_wait(&empty_bar[s], ((i / kBulkStages) - 1u) & 1u)) {
            ok = false;
            break;
          }
          if (*reinterpret_cast<volatile uint32_t*>(&s_stop)) break;
        }
        uint8_t* base = smem + size_t(s) * kListStageBytes;
        const uint64_t e0 = tile * kBulkTile;
        const uint32_t k =
            search_tensor(e0, __ldg(tile_first + e0 / kTileElems), list.n_tensors, offsets);
        const GradTensor* gt = list.tensors + k;
        TileInfo info{};
        info.tensor = k;
        info.flags = __ldg(&gt->flags);
        info.mode = e0 + kBulkTile > __ldg(offsets + k + 1) ? kTileMany : kTileOne;
        uintptr_t from = 0;
        uint32_t bytes = 0;
        if (info.mode == kTileOne && !(info.flags & kGradPitched)) {
          const uint32_t size = elem_bytes(info.flags & kGradTypeMask);
          const uintptr_t lo = __ldg(reinterpret_cast<const unsigned long long*>(&gt->ptr));
          const uintptr_t hi = lo + __ldg(&gt->elements) * size;
          const uintptr_t a = lo + (e0 - __ldg(offsets + k)) * size;
          from = a & ~uintptr_t(15);
          info.shift = uint32_t(a - from);
          bytes = kBulkTile * size + (info.shift ? 16u : 0u);
          if (from >= lo && from + bytes <= hi) info.mode = kTileStaged;
        }
        infos[s] = info;
        const bool staged = info.mode == kTileStaged;
        mbar_arrive_expect_tx(&full_bar[s], 3 * kListStateBytes + (staged ? bytes : 0u));
        if (staged) bulk_load(base, reinterpret_cast<const void*>(from), bytes, &full_bar[s]);
        bulk_load(base + kListGradBytes, master + e0, kListStateBytes, &full_bar[s]);
        bulk_load(base + kListGradBytes + kListStateBytes, mom + e0, kListStateBytes,
                  &full_bar[s]);
        bulk_load(base + kListGradBytes + 2 * kListStateBytes, var + e0, kListStateBytes,
                  &full_bar[s]);
      }
    }
  } else {
    const uint32_t t = threadIdx.x;
    pdl_wait();  // the decision is complete and visible
    if (t == 0) {
      s_go = (st->skipped == 0u && st->kernel_error == 0u) ? 1u : 0u;
      s_scale = st->loss_scale_used;
      s_clip = st->clip_apply;
      if (!s_go) s_stop = 1u;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kBulkConsumers) : "memory");
    if (!s_go) {
      // No update: take back the tiles the producer already started, so no copy
      // lands after the block exits.
      const uint32_t started = mine < kBulkStages ? uint32_t(mine) : kBulkStages;
      for (uint32_t u = 0; u < started; ++u) {
        ok &= mbar_wait(&full_bar[u], 0u);
        __syncwarp();
        if ((t & 31) == 0) mbar_arrive(&empty_bar[u]);
      }
    } else {
      const ScaleInfo sc = decode_scale(s_scale);
      const float clip = s_clip;
      ok = sc.mul ? list_consume<true>(smem, infos, full_bar, empty_bar, n_full, list, master,
                                       mom, var, w16, offsets, decay, p, sc, clip, bad)
                  : list_consume<false>(smem, infos, full_bar, empty_bar, n_full, list, master,
                                        mom, var, w16, offsets, decay, p, sc, clip, bad);
      // Ragged tail after the last whole tile: element by element, block 0.
      if (blockIdx.x == 0) {
        for (uint64_t e = n_full * kBulkTile + t; e < n; e += kBulkConsumers) {
          const uint32_t k =
              search_tensor(e, __ldg(tile_first + e / kTileElems), list.n_tensors, offsets);
          const float wd = __ldg(decay + k) ? p.decay_weight : p.no_decay_weight;
          const float x = grad_at(list.tensors, k, e - __ldg(offsets + k));
          const float gv = clipped(x, sc, clip);
          float m = mom[e], v = var[e];
          const float t1 = adamw_elem(master[e], gv, m, v, wd, p, bad);
          master[e] = t1;
          mom[e] = m;
          var[e] = v;
          w16[e] = bf16_rne_bits(t1);
        }
      }
    }
  }
  // After an expired wait the producer waits (bounded) for the tiles it still
  // has in flight, so no copy lands in shared memory after the block exits.
  if (__syncthreads_or(ok ? 0 : 1) && threadIdx.x == kBulkConsumers)
    for (uint32_t u = i > kBulkStages ? i - kBulkStages : 0u; u < i; ++u)
      mbar_wait(&full_bar[u % kBulkStages], (u / kBulkStages) & 1u);
  if (!ok) atomicOr(&st->kernel_error, 1u);
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
  const uint64_t skip = (t.flags & kGradPitched)
                            ? 0u
                            : uint64_t(units[i].index) * unit_elems *
                                  elem_bytes(t.flags & kGradTypeMask);
  units[i].ptr = static_cast<const uint8_t*>(t.ptr) + skip;
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

cudaError_t launch_list_norm(const GradListView& list, float scale, const DeviceScaler* scaler,
                             const GradPartials& part, cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  list_norm_kernel<<<list.n_units, kListThreads, 0, stream>>>(list, scale, scaler, part);
  return cudaGetLastError();
}

cudaError_t launch_list_finalize(const GradListView& list, const GradPartials& part, float scale,
                                 float max_norm, int kind, const GradListOut& out,
                                 cudaStream_t stream) {
  const uint32_t grid = 1u + (out.tensor_norms || out.tensor_max ? list.n_tensors : 0u);
  return launch_chained(list_finalize_kernel, grid, kFinalThreads, 0, stream, list, part, scale,
                        max_norm, kind, out);
}

cudaError_t launch_list_decide(const GradListView& list, const GradPartials& part,
                               DeviceScaler* scaler, DeviceStepState* st,
                               const FinalizeParams& fp, cudaStream_t stream) {
  return launch_chained(list_decide_kernel, 1u, kFinalThreads, 0, stream, list, part, scaler, st,
                        fp);
}

cudaError_t launch_list_clip(const GradListView& list, const GradListView& out, float scale,
                             const float* result, bool in_place, cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  return launch_chained(list_clip_kernel, list.n_units, kListThreads, 0, stream, list, out, scale,
                        result, in_place);
}

cudaError_t launch_list_accumulate(const GradListView& list, float* acc, int overwrite,
                                   cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  list_accumulate_kernel<<<list.n_units, kListThreads, 0, stream>>>(list, acc, overwrite);
  return cudaGetLastError();
}

cudaError_t launch_list_accumulate_norm(const GradListView& list, float* acc, int overwrite,
                                        float scale, const DeviceScaler* scaler,
                                        const GradPartials& part, cudaStream_t stream) {
  if (list.n_units == 0) return cudaSuccess;
  list_accumulate_norm_kernel<<<list.n_units, kListThreads, 0, stream>>>(list, acc, overwrite,
                                                                         scale, scaler, part);
  return cudaGetLastError();
}

int list_update_grid(int device) {
  cudaFuncSetAttribute(list_update_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       int(list_update_smem()));
  int per_sm = 0, sms = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, list_update_kernel, kBulkThreads,
                                                    list_update_smem()) != cudaSuccess ||
      per_sm <= 0)
    per_sm = 1;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      sms <= 0)
    sms = 148;
  return sms * per_sm;
}

cudaError_t launch_list_update(const GradListView& list, float* master, float* moment,
                               float* variance, uint16_t* w16, const uint64_t* offsets,
                               const uint8_t* decay, const uint32_t* tile_first,
                               const AdamwParams& p, DeviceStepState* st, int grid,
                               cudaStream_t stream) {
  const uint64_t tiles = list.elements / kBulkTile;
  const uint32_t blocks = uint32_t(tiles == 0 ? 1 : (uint64_t(grid) < tiles ? uint64_t(grid) : tiles));
  return launch_chained(list_update_kernel, blocks, kBulkThreads, list_update_smem(), stream,
                        list, master, moment, variance, w16, offsets, decay, tile_first, p, st);
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
