// Logit adjustment before sampling (sm_100a): repetition / presence / frequency penalties, sparse biases and grammar
// masks, each row with its own parameters. The order and arithmetic of penalties and mask are aib_sample's (sampler.cu,
// after Constraint.apply, generation/constrain.py:146-148); the reference has no penalties or biases.
//
// A CTA takes one slice of one row. It copies the slice and masks it, as bits: most tokens need no more. Meanwhile it
// counts the row's prior ids that fall into the slice in shared memory (15 bits a token, the 16th says that the token has
// a bias). After the copy every entry of the lists that falls into the slice writes its token's adjusted logit, computed
// from the raw one; entries of the same token write the same value. In place they first read, then write, and clear the
// counts of what they have written. Bound by bytes; a slice is as long as the grid allows (four CTAs an SM), since every
// slice reads the whole of the row's lists.
// Slices are cut in a shifted index u = v + sh, where sh is the row's distance from a 16-byte boundary in elements, so
// that vector accesses are aligned whatever the row's start.
// Measured (B200): 256 rows of 151669 bf16 with a mask 26 us (6.1 TB/s), with 1000 prior ids and 300 biases a row too 42 us:
// while a CTA reads the raw logits of its listed tokens it has no data on its way. Tried and slower: those reads ahead of
// the copy (58 us, they miss L2), listed tokens written first and left out of the copy (50 us), counts looked up by the
// copy itself (265 us, the rare path is in every vector's way).
#include <algorithm>
#include <atomic>
#include "common.cuh"

namespace aib {
namespace adjust {

constexpr int kMaxPrior = 32767;  // counts are 15 bits
constexpr int kMaxBias = 1024;
constexpr int kDeep = 4;          // vectors of a thread that are on their way at once
constexpr uint32_t kBiased = 0x8000u;

template <typename E>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr int kSlice = 8192;  // elements of a slice at most: 32 KB of the row
  static constexpr float kOut = -INFINITY;
};
template <>
struct Vec<uint16_t> {
  static constexpr int N = 8;
  static constexpr int kSlice = 16384;
  static constexpr uint16_t kOut = 0xFF80;
};
AIB_DEV float to_f(float x) { return x; }
AIB_DEV float to_f(uint16_t x) { return bf16_to_f32(x); }
AIB_DEV void from_f(float x, float* o) { *o = x; }
AIB_DEV void from_f(float x, uint16_t* o) { *o = bf16_rn(x); }
// A vector's masked elements (bits 0) to -inf.
AIB_DEV void mask_out(uint4& x, uint32_t bits, float) {
  if (!(bits & 1)) x.x = 0xFF800000u;
  if (!(bits & 2)) x.y = 0xFF800000u;
  if (!(bits & 4)) x.z = 0xFF800000u;
  if (!(bits & 8)) x.w = 0xFF800000u;
}
AIB_DEV uint32_t mask_pair(uint32_t x, uint32_t bits) {
  const uint32_t keep = (bits & 1 ? 0x0000FFFFu : 0u) | (bits & 2 ? 0xFFFF0000u : 0u);
  return (x & keep) | (0xFF80FF80u & ~keep);
}
AIB_DEV void mask_out(uint4& x, uint32_t bits, uint16_t) {
  x = make_uint4(mask_pair(x.x, bits), mask_pair(x.y, bits >> 2), mask_pair(x.z, bits >> 4), mask_pair(x.w, bits >> 6));
}

// Loads that the compiler may not put off until their values are used (the lists' work lies between): the slice's data,
// read once, and the mask's words, which neighbours read too. 256 rows of 151669 bf16 with a mask alone: 32 us with plain
// loads, 26 us with these.
AIB_DEV uint4 load_now(const uint4* p) {
  uint4 x;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
  return x;
}
AIB_DEV uint32_t load_now(const uint32_t* p) {
  uint32_t x;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(x) : "l"(p));
  return x;
}

template <typename E, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    adjust_kernel(const E* logits, long long ld, E* out, long long out_ld, int V, const int32_t* __restrict__ prior,
                  long long prior_ld, int n_prior, const float* __restrict__ rep, const float* __restrict__ pres,
                  const float* __restrict__ freq, const int32_t* __restrict__ bias_ids, long long ids_ld,
                  const float* __restrict__ bias, long long bias_ld, int n_bias, const uint32_t* __restrict__ mask,
                  long long mask_ld, int slice) {
  constexpr int N = Vec<E>::N;
  extern __shared__ __align__(16) uint32_t sm[];
  uint32_t* cnt = sm;  // slice / 2 words: two tokens each
  uint32_t* twice = cnt + slice / 2;  // slice / 32 words: the token has several biases
  int* bid = reinterpret_cast<int*>(twice + slice / 32);
  float* bval = reinterpret_cast<float*>(bid + n_bias);
  pdl_wait();
  pdl_trigger();
  const long long b = blockIdx.y;
  logits += b * ld;
  out += b * out_ld;
  const int sh = static_cast<int>(reinterpret_cast<uintptr_t>(logits) / sizeof(E) % N);
  const bool same = reinterpret_cast<uintptr_t>(out) / sizeof(E) % N == sh;
  const int base = static_cast<int>(blockIdx.x * slice) - sh;  // token of the slice's place 0
  const uint32_t* mrow = mask ? mask + b * mask_ld : nullptr;
  // Whole vectors [kbeg, kend) of the slice (none if logits and out lie differently). A thread's vectors are whole words
  // of the mask apart, so its place in a word is always the same.
  const int v0 = max(0, base), v1 = min(V, base + slice);
  const int kbeg = base < 0 ? N : 0, kend = same ? (v1 - base) / N * N : 0;
  auto whole = [&](int k) { return k < kend && k >= kbeg; };
  const int at = threadIdx.x * N;
  constexpr int kStep = kThreads * N;
  static_assert(kStep % 32 == 0, "whole words of the mask from one vector of a thread to the next");
  const uint4* src = reinterpret_cast<const uint4*>(logits + base + at);
  uint4* dst = reinterpret_cast<uint4*>(out + base + at);
  const uint32_t* words = mrow + ((base + at) >> 5);
  const int shift = (base + at) & 31;
  const bool two = shift + N > 32;
  uint4 x[kDeep];
  uint32_t lo[kDeep], hi[kDeep];
  auto load = [&](int k) {  // the thread's vectors from place k on, and their mask words
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      if (whole(k + j * kStep)) {
        x[j] = load_now(src + (k - at) / N + j * kThreads);
        if (mrow) {
          lo[j] = load_now(words + (k - at) / 32 + j * (kStep / 32));
          if (two) hi[j] = load_now(words + (k - at) / 32 + j * (kStep / 32) + 1);
        }
      }
    }
  };
  load(at);

  // ---- counts of the slice's tokens. The lists' first entries are on their way before the table is clear.
  constexpr int kItems = kThreads == 512 ? 8 : 4;  // entries of a thread at once: groups of four neighbours
  const int32_t* pr = prior + b * prior_ld;
  const int32_t* ids = bias_ids + b * ids_ld;
  const bool quad = !(reinterpret_cast<uintptr_t>(pr) & 15);
  int id[kItems];
  auto entries = [&](int i0) {  // the thread's entries of the prior list, from group i0 on
#pragma unroll
    for (int g = 0; g < kItems / 4; ++g) {
      const int i = (i0 + g * kThreads + threadIdx.x) * 4;
      int4 e = make_int4(-1, -1, -1, -1);
      if (quad && i + 4 <= n_prior) {
        e = *reinterpret_cast<const int4*>(pr + i);
      } else {
        if (i < n_prior) e.x = pr[i];
        if (i + 1 < n_prior) e.y = pr[i + 1];
        if (i + 2 < n_prior) e.z = pr[i + 2];
        if (i + 3 < n_prior) e.w = pr[i + 3];
      }
      id[4 * g] = e.x, id[4 * g + 1] = e.y, id[4 * g + 2] = e.z, id[4 * g + 3] = e.w;
    }
  };
  const float r = rep ? rep[b] : 1.0f, p = pres ? pres[b] : 0.0f, f = freq ? freq[b] : 0.0f;
  const bool penal = n_prior > 0 && (r != 1.0f || p != 0.0f || f != 0.0f);
  const int groups = penal ? (n_prior + 3) / 4 : 0;
  auto inside = [&](int t) { return t >= v0 && t < v1; };
  if (penal || n_bias > 0) {
    entries(0);
    constexpr int kFirst = 512 / kThreads;  // biases of a thread that are on their way already
    int b_id[kFirst];
    float b_val[kFirst];
#pragma unroll
    for (int j = 0; j < kFirst; ++j) {
      const int i = threadIdx.x + j * kThreads;
      b_id[j] = i < n_bias ? ids[i] : -1;
      b_val[j] = i < n_bias ? bias[b * bias_ld + i] : 0.0f;
    }
    for (int i = threadIdx.x; i < slice / 8 + slice / 128; i += kThreads)
      reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = 0; i0 < groups; i0 += kThreads * kItems / 4) {
      if (i0 > 0) entries(i0);
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        if (inside(id[i])) atomicAdd(&cnt[(id[i] - base) >> 1], 1u << (16 * ((id[i] - base) & 1)));
    }
    auto put = [&](int i, int t, float val) {
      const int k = t - base;
      bid[i] = t;
      bval[i] = val;
      if (inside(t)) {
        const uint32_t flag = kBiased << (16 * (k & 1));
        if (atomicOr(&cnt[k >> 1], flag) & flag) atomicOr(&twice[k >> 5], 1u << (k & 31));
      }
    };
#pragma unroll
    for (int j = 0; j < kFirst; ++j)
      if (static_cast<int>(threadIdx.x) + j * kThreads < n_bias) put(threadIdx.x + j * kThreads, b_id[j], b_val[j]);
    for (int i = threadIdx.x + 512; i < n_bias; i += kThreads) put(i, ids[i], bias[b * bias_ld + i]);
  }

  // ---- copy and mask
  for (int k = at; k < kend; k += kDeep * kStep) {
    if (k != at) load(k);
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      if (whole(k + j * kStep)) {
        if (mrow) mask_out(x[j], __funnelshift_r(lo[j], two ? hi[j] : 0, shift), E());
        dst[(k - at) / N + j * kThreads] = x[j];
      }
    }
  }
  auto one = [&](int v) {
    const E e = logits[v];
    out[v] = mrow && !(mrow[v >> 5] >> (v & 31) & 1) ? Vec<E>::kOut : e;
  };
  if (kbeg < kend) {  // what the row's start and end cut off
    if (v0 + static_cast<int>(threadIdx.x) < base + kbeg) one(v0 + threadIdx.x);
    if (base + kend + static_cast<int>(threadIdx.x) < v1) one(base + kend + threadIdx.x);
  } else {
#pragma unroll 4
    for (int v = v0 + static_cast<int>(threadIdx.x); v < v1; v += kThreads) one(v);
  }

  // ---- the tokens of the lists
  if (!penal && n_bias == 0) return;
  __syncthreads();
  const bool in_place = out == logits;
  auto count_of = [&](int t) -> uint32_t {  // 0 also for a token outside the slice
    return inside(t) ? reinterpret_cast<const uint16_t*>(cnt)[t - base] : 0;
  };
  auto allowed = [&](int t) { return !mrow || (mrow[t >> 5] >> (t & 31) & 1); };
  auto penalised = [&](float z, uint32_t c) {
    if (c) {
      z = z < 0.0f ? __fmul_rn(z, r) : __fdiv_rn(z, r);
      z = __fsub_rn(z, __fadd_rn(__fmul_rn(static_cast<float>(c), f), p));
    }
    return z;
  };
  // A round takes a thread's groups of prior ids and two biases: all that they read is on its way before anything is
  // written (in place nothing may be written before everything is read).
  constexpr int kBiases = 2;
  constexpr int kGroups = kItems / 4 * kThreads;  // groups of a round
  for (int round = 0; round * kGroups < groups || round * kThreads * kBiases < n_bias; ++round) {
    if (groups > kGroups) entries(round * kGroups);  // (a single round's are still there from the counting)
    uint32_t c[kItems], cb[kBiases];
    float z[kItems], zb[kBiases];
    int tb[kBiases];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      c[i] = round * kGroups < groups ? count_of(id[i]) : 0;
      if (c[i] & kBiased) c[i] = 0;  // the biases' entries see to it
    }
#pragma unroll
    for (int j = 0; j < kBiases; ++j) {
      const int i = (round * kBiases + j) * kThreads + threadIdx.x;
      tb[j] = i < n_bias ? bid[i] : -1;
      cb[j] = count_of(tb[j]);  // 0 for a token that an earlier round has written
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) z[i] = c[i] ? to_f(logits[id[i]]) : 0.0f;
#pragma unroll
    for (int j = 0; j < kBiases; ++j) zb[j] = cb[j] ? to_f(logits[tb[j]]) : 0.0f;
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (c[i] && !allowed(id[i])) c[i] = 0;
    if (in_place) __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (c[i]) {
        from_f(penalised(z[i], c[i]), &out[id[i]]);
        if (in_place) reinterpret_cast<uint16_t*>(cnt)[id[i] - base] = 0;
      }
    }
#pragma unroll
    for (int j = 0; j < kBiases; ++j) {
      const int t = tb[j];
      if (!cb[j]) continue;
      if (allowed(t)) {
        float s = bval[(round * kBiases + j) * kThreads + threadIdx.x];
        if (twice[(t - base) >> 5] >> ((t - base) & 31) & 1) {  // in the order of the list
          s = 0.0f;
          for (int i = 0; i < n_bias; ++i)
            if (bid[i] == t) s += bval[i];
        }
        from_f(penalised(zb[j], cb[j] & ~kBiased) + s, &out[t]);
      }
      if (in_place) reinterpret_cast<uint16_t*>(cnt)[t - base] = 0;
    }
    if (in_place) __syncthreads();
  }
}

template <typename E>
static int go(const void* logits, long long ld, void* out, long long out_ld, int B, int V, const int32_t* prior,
              long long prior_ld, int n_prior, const float* rep, const float* pres, const float* freq,
              const int32_t* bias_ids, long long ids_ld, const float* bias, long long bias_ld, int n_bias,
              const int32_t* mask, long long mask_ld, cudaStream_t s) {
  const int N = Vec<E>::N, span = V + N - 1;
  // Slices of a row: four CTAs an SM if there is that much, within 1024 .. kSlice elements each. Where that is all there is,
  // the CTAs are of 512 threads, since the slice with the most listed tokens decides (16 rows of 151936 with 4096 prior
  // ids each: 9.8 us, with 256 threads 14 us); more CTAs do better at 256 (256 rows: 42 us, with 512 threads 52 us).
  const int want = (4 * sm_count() + B - 1) / B;
  int slice = (span + want - 1) / want;
  slice = std::max(1024, std::min(Vec<E>::kSlice, (slice + 1023) / 1024 * 1024));
  const size_t smem = static_cast<size_t>(slice) * 2 + slice / 8 + static_cast<size_t>(n_bias) * 8;
  const dim3 grid((span + slice - 1) / slice, B);
  auto run = [&](auto kernel, int threads, std::atomic<uint64_t>& raised) {
    int dev = 0;  // the shared-memory limit is raised once on each device
    cudaGetDevice(&dev);
    if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
      const int rc = allow_smem(kernel, Vec<E>::kSlice * 2 + Vec<E>::kSlice / 8 + kMaxBias * 8);
      if (rc) return rc;
      if (dev < 64) raised.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch(kernel, grid, dim3(threads), smem, s, "aib_adjust_logits", static_cast<const E*>(logits), ld,
                  static_cast<E*>(out), out_ld, V, prior, prior_ld, n_prior, rep, pres, freq, bias_ids, ids_ld, bias,
                  bias_ld, n_bias, reinterpret_cast<const uint32_t*>(mask), mask_ld, slice);
  };
  static std::atomic<uint64_t> raised[2];
  if (static_cast<long long>(grid.x) * B <= 4LL * sm_count()) return run(adjust_kernel<E, 512>, 512, raised[0]);
  return run(adjust_kernel<E, 256>, 256, raised[1]);
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
  if (!aligned(es, logits, out) ||
      !aligned(4, prior, repetition, presence, frequency, bias_ids, bias, mask))
    return fail(AIB_EINVAL, "aib_adjust_logits: every argument must be aligned to its elements");
  const long long row = static_cast<long long>(V * es);
  const Rows2 in{reinterpret_cast<uintptr_t>(logits), row, {B, 1}, {ld, 0}, es},
      to{reinterpret_cast<uintptr_t>(out), row, {B, 1}, {out_ld, 0}, es};
  if (!(out == logits && (B == 1 || ld == out_ld)) && rows_meet(in, to))
    return fail(AIB_EINVAL, "aib_adjust_logits: out must be logits itself (with the same row stride) or share no memory with it");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? adjust::go<float>(logits, ld, out, out_ld, B, V, prior, prior_ld, n_prior, repetition, presence,
                                        frequency, bias_ids, bias_ids_ld, bias, bias_ld, n_bias, mask, mask_ld, s)
                    : adjust::go<uint16_t>(logits, ld, out, out_ld, B, V, prior, prior_ld, n_prior, repetition,
                                           presence, frequency, bias_ids, bias_ids_ld, bias, bias_ld, n_bias, mask,
                                           mask_ld, s);
}

}  // extern "C"
