// Device functions shared by the kernels of the step (kernels.cu) and of
// gradient lists (gradlist.cu): unscaling, the fixed f64 fold, the clip / skip
// decision, one AdamW element, mbarrier and bulk-copy primitives, programmatic
// dependent launch.
#pragma once

#include "slmopt_internal.h"

namespace slmopt {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ bool finite_f32(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Unscaling by s.  When s is a normal power of two whose reciprocal is also
// normal, x * (1/s) and x / s are the same exact real rounded once, so the
// multiply is bit-identical to the reference's true division; otherwise the
// IEEE division is used.
struct ScaleInfo {
  float s;
  float inv;
  bool mul;
};

__device__ __forceinline__ ScaleInfo decode_scale(float s) {
  const uint32_t b = __float_as_uint(s);
  const uint32_t e = (b >> 23) & 0xffu;
  ScaleInfo r;
  r.s = s;
  r.mul = ((b & 0x807fffffu) == 0u) && e >= 1u && e <= 253u;
  r.inv = __uint_as_float(((254u - e) & 0xffu) << 23);
  return r;
}

template <bool kMul>
__device__ __forceinline__ float unscale(float x, const ScaleInfo& sc) {
  if constexpr (kMul) {
    return __fmul_rn(x, sc.inv);
  } else {
    return __fdiv_rn(x, sc.s);
  }
}

__device__ __forceinline__ uint16_t bf16_rne_bits(float v) {
  // src/model/oracle.rs:300-304: bits + 0x7fff + lowest kept bit, keep the top half.
  const uint32_t b = __float_as_uint(v);
  return static_cast<uint16_t>((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
}

// ---- gradient loads (8 elements as f32) ------------------------------------
__device__ __forceinline__ void unpack_bf16x8(const uint4 r, float (&x)[8]) {
  x[0] = __uint_as_float(r.x << 16);
  x[1] = __uint_as_float(r.x & 0xffff0000u);
  x[2] = __uint_as_float(r.y << 16);
  x[3] = __uint_as_float(r.y & 0xffff0000u);
  x[4] = __uint_as_float(r.z << 16);
  x[5] = __uint_as_float(r.z & 0xffff0000u);
  x[6] = __uint_as_float(r.w << 16);
  x[7] = __uint_as_float(r.w & 0xffff0000u);
}

// ---- the fixed f64 tree -----------------------------------------------------
// Folds one double per thread of a 256-thread block; result valid in thread 0.
__device__ __forceinline__ double block_fold(double v, double* warp_sums) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = __dadd_rn(v, __shfl_down_sync(kFull, v, off));
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  if (lane == 0) warp_sums[warp] = v;
  __syncthreads();
  double r = 0.0;
  if (threadIdx.x == 0) {
    double w[kTreeThreads / 32];
#pragma unroll
    for (int i = 0; i < int(kTreeThreads / 32); ++i) w[i] = warp_sums[i];
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) {
#pragma unroll
      for (int i = 0; i < off; ++i) w[i] = __dadd_rn(w[i], w[i + off]);
    }
    r = w[0];
  }
  __syncthreads();
  return r;
}

// One 8-element vector's contribution to a tree lane: the values are
// unscaled, squared in f32, the 8 squares added pairwise in f32
// ((q0+q1)+(q2+q3))+((q4+q5)+(q6+q7)), and that sum added to the lane's f64
// accumulator.  Every term is >= 0, so the relative error of the partial stays
// below ~2.4e-7 (4 f32 roundings); one f32 -> f64 conversion per 8 elements
// keeps the conversion pipe off the critical path.  A non-finite or
// overflowing value makes the sum non-finite.
template <bool kMul>
__device__ __forceinline__ double add_squares8(double acc, float (&x)[8], const ScaleInfo& sc) {
  float q[kVec];
#pragma unroll
  for (uint32_t j = 0; j < kVec; ++j) {
    const float u = unscale<kMul>(x[j], sc);
    q[j] = __fmul_rn(u, u);
  }
  const float p = __fadd_rn(__fadd_rn(__fadd_rn(q[0], q[1]), __fadd_rn(q[2], q[3])),
                            __fadd_rn(__fadd_rn(q[4], q[5]), __fadd_rn(q[6], q[7])));
  return __dadd_rn(acc, static_cast<double>(p));
}

// The step's decision from the reduced sum: clip, skip / reject, and the
// dynamic scaler's next state.
struct StepDecision {
  float clip;        // min(max_norm / sqrtf((float)sum), 1); 1 for a zero sum; 0 if non-finite
  float clip_apply;  // what the update multiplies by
  float next_scale;
  uint32_t good;
  uint32_t skipped, rejected;
  int32_t status;
};

__device__ __forceinline__ StepDecision decide_step(double sum, uint32_t nonfinite, float scale,
                                                    uint32_t good_in, const FinalizeParams& fp) {
  StepDecision d;
  const float sumf = __double2float_rn(sum);
  const bool norm_bad = !finite_f32(sumf);
  if (norm_bad) {
    d.clip = 0.0f;
  } else if (sumf == 0.0f) {
    d.clip = 1.0f;
  } else {
    d.clip = __fdiv_rn(fp.max_grad_norm, __fsqrt_rn(sumf));
    d.clip = d.clip < 1.0f ? d.clip : 1.0f;
  }
  d.clip_apply = fp.apply_clip ? d.clip : 1.0f;
  d.skipped = 0u;
  d.rejected = 0u;
  d.status = kStatusOk;
  d.next_scale = scale;
  d.good = fp.dynamic ? good_in : 0u;
  if (nonfinite || norm_bad) {
    d.skipped = 1u;
    if (fp.nonfinite_policy == 1)
      d.status = nonfinite ? kStatusGradientNonfinite : kStatusNormNonfinite;
    if (fp.dynamic) {
      d.next_scale = __fmul_rn(scale, 0.5f);
      d.good = 0u;
    }
  } else if (fp.min_clip_accept > 0.0f && d.clip < fp.min_clip_accept) {
    d.skipped = 1u;
    d.rejected = 1u;
    d.status = kStatusGradientInvalid;
  } else if (fp.dynamic) {
    d.good += 1u;
    if (d.good >= fp.growth_interval) {
      d.next_scale = __fmul_rn(scale, 2.0f);
      d.good = 0u;
    }
  }
  return d;
}

// Publishes a decision: the step record and, for a dynamic scale, the scaler.
// result_nonfinite is left alone: the update kernels raise it, and it is
// cleared before they start.
__device__ __forceinline__ void write_decision(const StepDecision& d, double sum, uint32_t nonfinite,
                                               float scale, DeviceStepState* st,
                                               DeviceScaler* scaler, const FinalizeParams& fp) {
  st->sum_squares = sum;
  st->grad_norm = __dsqrt_rn(sum);
  st->clip_scale = d.clip;
  st->clip_apply = d.clip_apply;
  st->loss_scale_used = scale;
  st->nonfinite = nonfinite;
  st->rejected = d.rejected;
  st->skipped = d.skipped;
  st->status = d.status;
  if (fp.dynamic) {
    scaler->scale = d.next_scale;
    scaler->good_steps = d.good;
  }
  st->next_loss_scale = d.next_scale;
  st->good_steps = d.good;
}

__device__ __forceinline__ float adamw_elem(float th, float gv, float& m, float& v, float wd,
                                            const AdamwParams& p, bool& bad) {
  const float m1 = __fadd_rn(__fmul_rn(p.beta1, m), __fmul_rn(p.omb1, gv));
  const float v1 = __fadd_rn(__fmul_rn(p.beta2, v), __fmul_rn(__fmul_rn(p.omb2, gv), gv));
  const float mh = __fdiv_rn(m1, p.bc1);
  const float vh = __fdiv_rn(v1, p.bc2);
  const float den = __fadd_rn(__fsqrt_rn(vh), p.eps);
  const float upd = __fadd_rn(__fdiv_rn(mh, den), __fmul_rn(wd, th));
  const float t1 = __fsub_rn(th, __fmul_rn(p.lr, upd));
  bad |= !(finite_f32(m1) && finite_f32(v1) && finite_f32(t1));
  m = m1;
  v = v1;
  return t1;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Waits for the phase with the given parity; false after ~4 s.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 255u) == 0u && global_ns() - t0 > 4000000000ull) return false;
  }
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void lds4(const float* p, float (&x)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
}

// Programmatic dependent launch: the norm pass lets the update grid launch
// while its own blocks are still running; the update's producer warps start
// streaming tiles at once (the norm pass writes none of g / master / m / v),
// and its consumers wait for the norm pass to complete before they read the
// step's decision.  Without the launch attribute (or after a kernel that does
// not trigger) the wait returns at once.
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace
}  // namespace slmopt
