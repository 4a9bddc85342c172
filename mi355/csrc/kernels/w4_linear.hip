// Products of a few rows with 4-bit weights:  y[m,n] = sum_k x[m,k] * w[n,k],
// w[n,k] = e2m1(code[n,k]) * 2^(exp[n, k/32] - 127).
//
// Codes are two a byte (low nibble: even k), row-major (N, K/2), one exponent
// byte for 32 inputs (N, K/32): 4.25 bits a weight, laid out as the checkpoint
// holds them.  With few rows the weight bytes bound the product, so every
// weight is read once from memory, straight into registers, 16 bytes a lane:
// lane (n = lane%16, g = lane/16) owns the 32 codes of ONE scale group, row n,
// k = 128c + 32g .. +32.  CDNA4 converts two codes with a per-lane power-of-two
// scale in one instruction, so the group scale costs nothing, and the order of
// k inside a matrix instruction is free, so MFMA i takes bytes 4i..4i+3 of each
// lane (k = 128c + 32g + 8i + j) and x is read at the same k: no shuffle.
//
// Roundings: a converted weight has 2 significant bits and is exact in bf16 and
// fp16.  Its exponent is taken relative to the row's largest group exponent
// (put back in 32 bits at the end), so that fp16 holds it exactly down to
// 2^-23 of the row's largest scale; below that it is less than half a unit of
// an fp32 sum.  Sums are fp32; y is rounded once.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "../common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

template <typename T> struct Frag;
template <> struct Frag<__hip_bfloat16> {
  using vec = bf16x8;
  template <int S> static DEVINL unsigned cvt2(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, S));
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Frag<__half> {
  using vec = f16x8;
  template <int S> static DEVINL unsigned cvt2(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, S));
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// eight codes of one scale group -> eight weights
template <typename T>
DEVINL typename Frag<T>::vec decode8(unsigned codes, float scale) {
  u32x4 r;
  r[0] = Frag<T>::template cvt2<0>(codes, scale);
  r[1] = Frag<T>::template cvt2<1>(codes, scale);
  r[2] = Frag<T>::template cvt2<2>(codes, scale);
  r[3] = Frag<T>::template cvt2<3>(codes, scale);
  return __builtin_bit_cast(typename Frag<T>::vec, r);
}

// 2^(e - row_e) as a float; differences under 2^-100 count as 2^-100
DEVINL float group_scale(int e, int row_e) {
  const int d = max(e - row_e, -100);
  return __builtin_bit_cast(float, (unsigned)(d + 127) << 23);
}

// ---------------------------------------------------------------------------
// Up to 16*MT rows, x straight from the caches: one wave owns 16 outputs and
// every WAVES-th 128-wide piece of K, the block's waves are summed through LDS
// in wave order (the same sum every time).
// ---------------------------------------------------------------------------
template <typename T, int MT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
w4_few_rows(const T* __restrict__ x, const unsigned char* __restrict__ codes,
            const unsigned char* __restrict__ exps, const unsigned char* __restrict__ row_exp,
            T* __restrict__ y, int M, int N, int K, long ldx) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c16 = lane & 15;
  const int n = blockIdx.x * 16 + c16;
  const int m0 = blockIdx.y * (16 * MT);
  const bool n_ok = n < N;
  const int row_e = n_ok ? row_exp[n] : 127;
  const unsigned char* crow = codes + (long)(n_ok ? n : 0) * (K >> 1);
  const unsigned char* erow = exps + (long)(n_ok ? n : 0) * (K >> 5);

  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int k0 = wave * 128; k0 < K; k0 += WAVES * 128) {
    const int k = k0 + 32 * g;
    const bool k_ok = k < K;              // K is a multiple of 32
    u32x4 w = u32x4{0u, 0u, 0u, 0u};
    float scale = 1.f;
    if (k_ok && n_ok) {
      w = *reinterpret_cast<const u32x4*>(crow + (k >> 1));
      scale = group_scale(erow[k >> 5], row_e);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const typename Frag<T>::vec wf = decode8<T>(w[i], scale);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int m = m0 + 16 * t + c16;
        u32x4 xv = u32x4{0u, 0u, 0u, 0u};
        if (k_ok && m < M) xv = *reinterpret_cast<const u32x4*>(x + m * ldx + k + 8 * i);
        acc[t] = Frag<T>::mfma(__builtin_bit_cast(typename Frag<T>::vec, xv), wf, acc[t]);
      }
    }
  }

  __shared__ f32x4 part[WAVES][MT][64];
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // D layout: column n = lane%16, row m = 4*(lane/16) + r
  // 2^(row_e - 127); byte 0 is the subnormal 2^-127
  const float back = __builtin_bit_cast(float, row_e ? (unsigned)row_e << 23 : 0x00400000u);
  for (int t = wave; t < MT; t += WAVES) {
    f32x4 s = part[0][t][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) {
      const f32x4 p = part[v][t][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] += p[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + 16 * t + 4 * g + r;
      if (n_ok && m < M) y[(long)m * N + n] = DT<T>::from_f32(s[r] * back);
    }
  }
}

}  // namespace

torch::Tensor w4_linear(torch::Tensor x, torch::Tensor codes, torch::Tensor exps,
                        torch::Tensor row_exp) {
  TORCH_CHECK(x.dim() == 2 && codes.dim() == 2 && exps.dim() == 2 && row_exp.dim() == 1,
              "w4_linear: x (M,K), codes (N,K/2), exps (N,K/32), row_exp (N)");
  const long M = x.size(0), K = x.size(1), N = codes.size(0);
  TORCH_CHECK(K > 0 && K % 32 == 0 && codes.size(1) * 2 == K && exps.size(0) == N &&
                  exps.size(1) * 32 == K && row_exp.size(0) == N,
              "w4_linear: x has ", K, " inputs, codes ", codes.size(1) * 2, ", exps ",
              exps.size(1) * 32);
  // 65535 blocks of 64 rows
  TORCH_CHECK(M < (1L << 22) - 64 && N < (1L << 31) && K < (1L << 30), "w4_linear: too large");
  for (const auto& t : {codes, exps, row_exp})
    TORCH_CHECK(t.scalar_type() == torch::kByte && t.is_contiguous() && t.device() == x.device(),
                "w4_linear: codes and exponents must be contiguous uint8 on x's device");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
              "w4_linear: codes must be 16-byte aligned");
  c10::DeviceGuard guard(x.device());
  auto y = torch::empty({M, N}, x.options());
  if (M == 0 || N == 0) return y;
  // rows of x are read 16 bytes at a time
  if (x.stride(1) != 1 || x.stride(0) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0)
    x = x.clone(at::MemoryFormat::Contiguous);
  auto stream = at::hip::getCurrentHIPStream().stream();
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const dim3 grid((N + 15) / 16, M <= 16 ? 1 : (M + 63) / 64);
    auto call = [&](auto kernel, int waves) {
      hipLaunchKernelGGL(kernel, grid, dim3(waves * 64), 0, stream, (const T*)x.data_ptr(),
                         codes.data_ptr<unsigned char>(), exps.data_ptr<unsigned char>(),
                         row_exp.data_ptr<unsigned char>(), (T*)y.data_ptr(), (int)M, (int)N,
                         (int)K, (long)x.stride(0));
    };
    if (M <= 16) call(w4_few_rows<T, 1, 8>, 8);
    else call(w4_few_rows<T, 4, 4>, 4);
  };
  if (x.scalar_type() == torch::kBFloat16) go(__hip_bfloat16());
  else if (x.scalar_type() == torch::kHalf) go(__half());
  else TORCH_CHECK(false, "w4_linear: bf16 or fp16 inputs, got ", x.scalar_type());
  HIP_CHECK_KERNEL();
  return y;
}
