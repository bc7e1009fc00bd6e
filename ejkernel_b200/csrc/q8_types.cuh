// The 8-bit cache: parameters of its kernels and the conversions of its codes.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ejk_q8.h"
#include "rpa_device.cuh"
#include "rpa_types.h"

namespace ejk {

// Where a row lives: kv_pages [P, Hkv, 2, page, D], kv_scales [P, Hkv, 2, page >> block_shift]
struct Q8Cache {
  uint8_t* pages;
  float* scales;
  int32_t num_pages, page_size, Hkv, D;
  int32_t block_shift;  // log2 of the tokens that share a scale
};

// Codes to f16, exactly, four at a time.  widen: bytes 0, 1 and 2, 3 of `w`; widen_interleaved: bytes 0, 2 and 1, 3.
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

struct CodeE4M3 {
  static __device__ __forceinline__ uint32_t widen2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)two));
    return r;
  }
  static __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = widen2(w);
    hi = widen2(w >> 16);
  }
  static __device__ __forceinline__ void widen_interleaved(uint32_t w, uint32_t& even, uint32_t& odd) {
    widen(prmt(w, w, 0x3120u), even, odd);
  }

  static constexpr float kMax = 448.f;
  static __device__ __forceinline__ float decode(uint8_t c) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"((uint16_t)c));
    return __half2float(__ushort_as_half((uint16_t)h));
  }
  // the nearest codes, ties to even, `a` in the low byte
  static __device__ __forceinline__ uint32_t encode2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(b), "f"(a));
    return r;
  }
  // biased exponent of the smallest power of two s with amax <= 448 * s: 448 = 1.75 * 2^8
  static __device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    return (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  }
};
struct CodeI8 {
  // byte + 128 under the exponent of 1024 is the f16 1152 + code; the difference is exact
  static __device__ __forceinline__ uint32_t less_1152(uint32_t w) {
    const uint32_t b = 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  static __device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = less_1152(prmt(w, 0x64646464u, 0x4140u));
    hi = less_1152(prmt(w, 0x64646464u, 0x4342u));
  }
  static __device__ __forceinline__ void widen_interleaved(uint32_t w, uint32_t& even, uint32_t& odd) {
    w ^= 0x80808080u;
    even = less_1152(prmt(w, 0x64646464u, 0x4240u));
    odd = less_1152(prmt(w, 0x64646464u, 0x4341u));
  }

  static constexpr float kMax = 127.f;
  static __device__ __forceinline__ float decode(uint8_t c) { return (float)(int8_t)c; }
  static __device__ __forceinline__ uint32_t encode2(float a, float b) {
    // 1.5 * 2^23 + x: the sum's low bits are x rounded to the nearest integer, ties to even
    return prmt(__float_as_uint(a + 12582912.f), __float_as_uint(b + 12582912.f), 0x0040u) & 0xffffu;
  }
  // 127 = 1.984375 * 2^6
  static __device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    return (int)(amax_bits >> 23) - 6 + ((amax_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  }
};
template <typename Code>
__device__ __forceinline__ float power_of_two_scale(float amax) {
  int e = Code::scale_exponent(__float_as_uint(amax));
  e = e < 1 ? 1 : e;  // not below 2^-126: scale and 1 / scale stay normal (amax < 2^128, so e <= 249)
  return __uint_as_float((uint32_t)e << 23);
}
// 1 / s of a power of two between 2^-126 and 2^126, exactly
__device__ __forceinline__ float power_of_two_inverse(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

// cap_log2 * tanh(t) as cap_log2 * (1 - 2 / (e^2t + 1)) is off by up to cap * 2^-22, which is an error of the logit: up to this cap it
// stays below 2^-12.  Beyond it small t go through tanh's series, t - t^3/3 + 2t^5/15 - 17t^7/315 + 62t^9/2835, whose next term is
// 1e-8 of the value at 1/4.  The pipelined kernels do not have that form (in line it cost every decode batch 1 to 7 %): such calls
// go to the simple one.
constexpr float kPlainCap = 1024.f;
__device__ __forceinline__ float soft_cap_large(float cap_log2, float t) {
  const float s = t * t;
  const float y = t + t * s * (-1.f / 3.f + s * (2.f / 15.f + s * (-17.f / 315.f + s * (62.f / 2835.f))));
  return cap_log2 * (fabsf(t) < 0.25f ? y : soft_cap_tanh(t));
}

// Offsets of a sequence that no kernel serves (they report it): its rows that there are, are zero.
__device__ __forceinline__ bool bad_rows(int q0, int q1, int T) { return q1 < q0 || q0 < 0 || q1 > T; }

// host side, shared by the entry points (defined in rpa_api.cu)
struct LaunchOptions {
  int min_chunk, prefill_rows, prefill_share, prefill_split, overlap, wait_ms, path, test_withhold;
};
LaunchOptions launch_options();
// SM count of the current device; 0: no device, or not an sm_100 one
int sm100_sm_count();
int check_rpa_shape(const ejk_rpa_shape& s);
void set_last_launches(int n);

// launchers
cudaError_t launch_q8_gather(const Params& p, const Q8Cache& c, int dtype, int code, cudaStream_t stream);
constexpr int kQ8TicketsPerCta = 12;  // arrival counters of the split-KV kernel: 3 per consumer warp
// the pipelined kernel: page sizes that are multiples of 8
bool q8_tma_supported(int page_size);
cudaError_t q8_tensor_map(CUtensorMap* map, const Q8Cache& c, int box_tokens);
cudaError_t launch_q8_splitkv(const Params& p, const Q8Cache& c, int dtype, int code, int n_sm, cudaStream_t stream, bool pdl);
// tcgen05 tiles for sequences with many query rows (head_dim 64 and 128)
cudaError_t launch_q8_plan(const Params& p, int n_sm, cudaStream_t stream, bool pdl);
bool q8_prefill_supported(int head_dim);
cudaError_t launch_q8_prefill(const Params& p, const Q8Cache& c, int dtype, int code, int n_sm, cudaStream_t stream, bool pdl);
cudaError_t launch_q8_write(const void* keys, const void* values, long long key_stride, long long value_stride,
                            const Q8Cache& c, const int32_t* slots, int32_t* status, int rows, int dtype, int code,
                            cudaStream_t stream);
cudaError_t launch_q8_read(const Q8Cache& c, const int32_t* slots, void* keys, void* values, int32_t* status, int rows,
                           int dtype, int code, cudaStream_t stream);
constexpr int kPageTableMaxRows = 16384;  // three sums per row in shared memory
cudaError_t launch_page_tables(const int32_t* query_lens, const int32_t* context_lens, int32_t* tables, int32_t* free_pages,
                               const int32_t* num_free, const int32_t* num_seqs, const uint8_t* finished,
                               int32_t* new_lens, int32_t* starts, int32_t* slots, int32_t* new_free, int32_t* status,
                               int S, int pps, int page, int capacity, int T, cudaStream_t stream);

}  // namespace ejk
