// Logit adjustment before sampling (sm_100a): repetition / presence / frequency penalties, sparse biases and grammar
// masks, each row with its own parameters. The order and arithmetic of penalties and mask are aib_sample's (sampler.cu,
// after Constraint.apply, generation/constrain.py:146-148); the reference has no penalties or biases.
//
// A CTA takes one slice of one row: it counts the row's prior ids that fall into the slice in shared memory (16 bits a
// token), lists the slice's biases in their order, and then streams the slice once: read, adjust in fp32, write.
// Slices are cut in a shifted index u = v + sh, where sh is the row's distance from a 16-byte boundary in elements, so
// that vector accesses are aligned whatever the row's start.
#include "common.cuh"

namespace aib {
namespace adjust {

constexpr int kThreads = 256;
constexpr int kMaxPrior = 65535;  // counts are 16 bits
constexpr int kMaxBias = 1024;

template <typename E>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
};
template <>
struct Vec<uint16_t> {
  static constexpr int N = 8;
};
AIB_DEV float to_f(float x) { return x; }
AIB_DEV float to_f(uint16_t x) { return bf16_to_f32(x); }
AIB_DEV void from_f(float x, float* o) { *o = x; }
AIB_DEV void from_f(float x, uint16_t* o) { *o = bf16_rn(x); }

template <typename E>
__global__ void __launch_bounds__(kThreads)
    adjust_kernel(const E* logits, long long ld, E* out, long long out_ld, int V, const int32_t* __restrict__ prior,
                  long long prior_ld, int n_prior, const float* __restrict__ rep, const float* __restrict__ pres,
                  const float* __restrict__ freq, const int32_t* __restrict__ bias_ids, long long ids_ld,
                  const float* __restrict__ bias, long long bias_ld, int n_bias, const uint32_t* __restrict__ mask,
                  long long mask_ld, int slice) {
  constexpr int N = Vec<E>::N;
  extern __shared__ __align__(16) uint32_t sm[];
  uint32_t* cnt = sm;                        // slice / 2 words: two 16-bit counts each
  uint32_t* flag = cnt + slice / 2;          // slice / 32 words: the token has a bias
  int* bid = reinterpret_cast<int*>(flag + slice / 32);
  float* bval = reinterpret_cast<float*>(bid + n_bias);
  __shared__ int wsum[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < slice / 2 + slice / 32; i += kThreads) sm[i] = 0;
  pdl_wait();
  pdl_trigger();
  const long long b = blockIdx.y;
  logits += b * ld;
  out += b * out_ld;
  const int sh = static_cast<int>(reinterpret_cast<uintptr_t>(logits) / sizeof(E) % N);
  const int so = static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(E) % N);
  const int u0 = blockIdx.x * slice;
  const float r = rep ? rep[b] : 1.0f, p = pres ? pres[b] : 0.0f, f = freq ? freq[b] : 0.0f;
  const bool penal = n_prior > 0 && (r != 1.0f || p != 0.0f || f != 0.0f);
  __syncthreads();
  if (penal) {
    const int32_t* pr = prior + b * prior_ld;
    for (int i = threadIdx.x; i < n_prior; i += kThreads) {
      const int id = pr[i];
      const unsigned k = static_cast<unsigned>(id) + sh - u0;
      if (id >= 0 && id < V && k < static_cast<unsigned>(slice)) atomicAdd(&cnt[k >> 1], 1u << (16 * (k & 1)));
    }
  }
  int nb = 0;
  if (n_bias > 0) {  // the slice's biases, in the order of the list
    for (int i0 = 0; i0 < n_bias; i0 += kThreads) {
      const int i = i0 + threadIdx.x;
      int id = i < n_bias ? bias_ids[b * ids_ld + i] : -1;
      const unsigned k = static_cast<unsigned>(id) + sh - u0;
      const bool in = id >= 0 && id < V && k < static_cast<unsigned>(slice);
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (lane == 0) wsum[warp] = __popc(m);
      __syncthreads();
      int at = nb + __popc(m & ((1u << lane) - 1));
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += wsum[w];
        nb += wsum[w];
      }
      if (in) {
        bid[at] = static_cast<int>(k);
        bval[at] = bias[b * bias_ld + i];
        atomicOr(&flag[k >> 5], 1u << (k & 31));
      }
      __syncthreads();
    }
  }
  __syncthreads();
  const uint32_t* mrow = mask ? mask + b * mask_ld : nullptr;
  for (int k0 = threadIdx.x * N; k0 < slice; k0 += kThreads * N) {
    const int v0 = u0 + k0 - sh;
    if (v0 >= V) break;
    if (v0 + N <= 0) continue;
    const bool whole = v0 >= 0 && v0 + N <= V;
    alignas(16) E x[N];
    if (whole) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(logits + v0);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (v0 + i >= 0 && v0 + i < V) x[i] = logits[v0 + i];
    }
    alignas(16) E y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int v = v0 + i, k = k0 + i;
      if (v < 0 || v >= V) continue;
      float z = to_f(x[i]);
      if (penal) {
        const uint32_t c = (cnt[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
        if (c) {
          z = z < 0.0f ? __fmul_rn(z, r) : __fdiv_rn(z, r);
          z = __fsub_rn(z, __fadd_rn(__fmul_rn(static_cast<float>(c), f), p));
        }
      }
      if (nb > 0 && (flag[k >> 5] >> (k & 31) & 1)) {
        float s = 0.0f;
        for (int j = 0; j < nb; ++j)
          if (bid[j] == k) s += bval[j];
        z += s;
      }
      if (mrow && !(mrow[v >> 5] >> (v & 31) & 1)) z = -INFINITY;
      from_f(z, &y[i]);
    }
    if (whole && sh == so) {
      *reinterpret_cast<uint4*>(out + v0) = *reinterpret_cast<const uint4*>(y);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (v0 + i >= 0 && v0 + i < V) out[v0 + i] = y[i];
    }
  }
}

template <typename E>
static int go(const void* logits, long long ld, void* out, long long out_ld, int B, int V, const int32_t* prior,
              long long prior_ld, int n_prior, const float* rep, const float* pres, const float* freq,
              const int32_t* bias_ids, long long ids_ld, const float* bias, long long bias_ld, int n_bias,
              const int32_t* mask, long long mask_ld, cudaStream_t s) {
  const int slice = 4096;
  const int N = Vec<E>::N;
  const size_t smem = slice * 2 + slice / 8 + static_cast<size_t>(n_bias) * 8;
  const dim3 grid((V + N - 1 + slice - 1) / slice, B);
  return launch(adjust_kernel<E>, grid, dim3(kThreads), smem, s, "aib_adjust_logits", static_cast<const E*>(logits), ld,
                static_cast<E*>(out), out_ld, V, prior, prior_ld, n_prior, rep, pres, freq, bias_ids, ids_ld, bias,
                bias_ld, n_bias, reinterpret_cast<const uint32_t*>(mask), mask_ld, slice);
}

}  // namespace adjust
}  // namespace aib

using namespace aib;

extern "C" {

int aib_adjust_logits(const void* logits, int64_t ld, void* out, int64_t out_ld, int dtype, int B, int V,
                      const int32_t* prior, int64_t prior_ld, int n_prior, const float* repetition,
                      const float* presence, const float* frequency, const int32_t* bias_ids, int64_t bias_ids_ld,
                      const float* bias, int64_t bias_ld, int n_bias, const int32_t* mask, int64_t mask_ld,
                      void* stream) {
  if (!logits || !out || B <= 0 || B > 65535 || V <= 0 || V > (1 << 30) || (dtype != 0 && dtype != 1) || n_prior < 0 ||
      n_bias < 0 || (n_prior > 0 && !prior) || (n_bias > 0 && (!bias_ids || !bias)) || ld < 0 || out_ld < 0 ||
      prior_ld < 0 || bias_ids_ld < 0 || bias_ld < 0 || mask_ld < 0 || (B > 1 && out_ld < V))
    return fail(AIB_EINVAL, "aib_adjust_logits: bad arguments");
  if (n_prior > adjust::kMaxPrior || n_bias > adjust::kMaxBias)
    return fail(AIB_ENOTSUP, "aib_adjust_logits: at most %d prior ids and %d biases a row (%d, %d)", adjust::kMaxPrior,
                adjust::kMaxBias, n_prior, n_bias);
  const size_t es = dtype == 0 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % es)
    return fail(AIB_EINVAL, "aib_adjust_logits: logits and out must be aligned to their elements");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? adjust::go<float>(logits, ld, out, out_ld, B, V, prior, prior_ld, n_prior, repetition, presence,
                                        frequency, bias_ids, bias_ids_ld, bias, bias_ld, n_bias, mask, mask_ld, s)
                    : adjust::go<uint16_t>(logits, ld, out, out_ld, B, V, prior, prior_ld, n_prior, repetition,
                                           presence, frequency, bias_ids, bias_ids_ld, bias, bias_ld, n_bias, mask,
                                           mask_ld, s);
}

}  // extern "C"
