// Paged key-value cache (sm_100a): appending new tokens with q/k norm and position rotation, and attention of one new
// token per sequence. No counterpart in the reference, whose caches are contiguous (core/engine.py:234-235); the
// arithmetic is that of qk_rope_cache_k and attn_k (kernels/tkernels.py:82-150).
//
// Sequence b's row at position p is row p % page of page table[b * table_ld + p / page] of the pool. Device data is
// checked where it is used: a position past the table's last page records AIB_DEV_BAD_POS, a page id outside the pool
// AIB_DEV_BAD_PAGE, and the row is neither written nor attended.
#include <algorithm>
#include "common.cuh"

namespace aib {
namespace paged {

struct Kv {
  uint16_t* k;
  uint16_t* v;
  long long page_stride, head_stride, row_stride;  // elements
  int pages, KV;
  int page_shift;  // rows per page = 1 << page_shift
};
// [T, heads, HD] rows: token and head strides in elements, inner stride 1; vec: pairs may be read as one word
template <typename E>
struct Rows {
  E* p;
  long long ts, hs;
  int vec;
};

// A pair of neighbouring elements (HD 128) or one element (HD 64) per lane as floats, and back.
template <int PER>
AIB_DEV void load_per(const float* p, int vec, float* o) {
  if (PER == 2 && vec) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    o[0] = t.x;
    o[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = p[i];
  }
}
template <int PER>
AIB_DEV void load_per(const uint16_t* p, int vec, float* o) {
  if (PER == 2 && vec) {
    const uint32_t t = *reinterpret_cast<const uint32_t*>(p);
    o[0] = __uint_as_float(t << 16);
    o[1] = __uint_as_float(t & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = bf16_to_f32(p[i]);
  }
}
template <int PER>
AIB_DEV void store_per(float* p, int vec, const float* o) {
  if (PER == 2 && vec) {
    *reinterpret_cast<float2*>(p) = make_float2(o[0], o[PER - 1]);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = o[i];
  }
}
template <int PER>
AIB_DEV void store_per(uint16_t* p, int vec, const float* o) {
  if (PER == 2 && vec) {
    *reinterpret_cast<uint32_t*>(p) = bf16x2_rn(o[0], o[PER - 1]);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = bf16_rn(o[i]);
  }
}

// cos and sin of p * inv. The product is formed in 64 bits (exact: 31 x 24 bits fit with at most one rounding in the
// last place) and reduced by whole turns there, so a far position loses nothing; a float product would be off by
// p * 2^-24 radians.
AIB_DEV void rotation(long long p, float inv, float* c, float* s) {
  const double a = static_cast<double>(p) * static_cast<double>(inv);
  const double n = rint(a * 0.15915494309189533577);
  const float r = static_cast<float>(fma(-n, 6.283185307179586477, a));
  sincosf(r, s, c);
}

// Largest b in [0, B) with cu[b] <= t (0 if none): the warp probes 32 places a round. cu is device data: whatever it
// holds, the result is in range.
AIB_DEV int find_seq(const int32_t* cu, int B, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, i < hi && cu[i] <= t);
    const int n = max(1, __popc(m));
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

constexpr int kAppWarps = 8;
constexpr int kAppBatch = 4;  // head vectors a warp holds at once

// One warp takes `per` of a token's head vectors (q heads, then k heads, then v heads); the lane holds dimensions
// r .. r + PER - 1 and their rotation partners HD/2 further, so norm and rotation need no exchange but the sum of
// squares, and the token's cosines and sines are computed once per warp.
template <int HD, typename E>
__global__ void __launch_bounds__(32 * kAppWarps)
    append_kernel(Kv c, const int32_t* __restrict__ table, int table_ld, int max_pages, const int64_t* __restrict__ pos,
                  const int32_t* __restrict__ cu, int B, int T, int H, Rows<const E> q, Rows<const E> k,
                  Rows<const E> v, Rows<E> qo, const uint16_t* __restrict__ qn, const uint16_t* __restrict__ kn,
                  const float* __restrict__ inv, float eps, int parts, int per) {
  constexpr int PER = HD / 64, HALF = HD / 2;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * kAppWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(w / parts);
  if (t >= T) return;
  int b = t, off = 0;
  if (cu) {
    if (t >= cu[B]) return;  // a row behind the last sequence
    b = find_seq(cu, B, t);
    off = t - cu[b];
    if (off < 0) return;
  }
  const long long p0 = pos[b], p = p0 + off;
  if (p0 < 0) return;  // an unused row of the batch
  const int r = lane * PER;
  float cs[PER], sn[PER];
  if (inv) {
#pragma unroll
    for (int i = 0; i < PER; ++i) rotation(p, inv[r + i], &cs[i], &sn[i]);
  }
  // where the token's k and v rows go
  const long long pg = p >> c.page_shift;
  long long row = -1;
  if (pg >= max_pages) {
    if (lane == 0) set_status(AIB_DEV_BAD_POS);
  } else {
    const int id = table[static_cast<long long>(b) * table_ld + pg];
    if (id < 0 || id >= c.pages) {
      if (lane == 0) set_status(AIB_DEV_BAD_PAGE);
    } else {
      row = id * c.page_stride + (p & ((1 << c.page_shift) - 1)) * c.row_stride;
    }
  }
  const int nv = H + 2 * c.KV, v0 = static_cast<int>(w % parts) * per, v1 = min(nv, v0 + per);
  for (int h0 = v0; h0 < v1; h0 += kAppBatch) {
    float x[kAppBatch][2 * PER];
#pragma unroll
    for (int i = 0; i < kAppBatch; ++i) {
      const int h = h0 + i;
      if (h >= v1) break;
      const E* src;
      int vec;
      if (h < H) {
        src = q.p + t * q.ts + h * q.hs;
        vec = q.vec;
      } else if (h < H + c.KV) {
        src = k.p + t * k.ts + (h - H) * k.hs;
        vec = k.vec;
      } else {
        src = v.p + t * v.ts + (h - H - c.KV) * v.hs;
        vec = v.vec;
      }
      load_per<PER>(src + r, vec, x[i]);
      load_per<PER>(src + r + HALF, vec, x[i] + PER);
    }
#pragma unroll
    for (int i = 0; i < kAppBatch; ++i) {
      const int h = h0 + i;
      if (h >= v1) break;
      float* a = x[i];
      float* z = x[i] + PER;
      const bool isq = h < H, isv = h >= H + c.KV;
      if (!isv) {
        const uint16_t* wn = isq ? qn : kn;
        if (wn) {
          float ss = 0.0f;
#pragma unroll
          for (int j = 0; j < 2 * PER; ++j) ss += x[i][j] * x[i][j];
          const float rs = rsqrtf(warp_sum(ss) / static_cast<float>(HD) + eps);
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            a[j] = bf16_to_f32(wn[r + j]) * (a[j] * rs);
            z[j] = bf16_to_f32(wn[r + j + HALF]) * (z[j] * rs);
          }
        }
        if (inv) {
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const float lo = a[j], hi = z[j];
            a[j] = lo * cs[j] - hi * sn[j];
            z[j] = hi * cs[j] + lo * sn[j];
          }
        }
      }
      if (isq) {
        E* dst = qo.p + t * qo.ts + h * qo.hs;
        store_per<PER>(dst + r, qo.vec, a);
        store_per<PER>(dst + r + HALF, qo.vec, z);
      } else if (row >= 0) {
        uint16_t* dst = isv ? c.v + row + (h - H - c.KV) * c.head_stride : c.k + row + (h - H) * c.head_stride;
        store_per<PER>(dst + r, 1, a);
        store_per<PER>(dst + r + HALF, 1, z);
      }
    }
  }
}

// ---------------------------------------------------------------------------------- attention
constexpr int GT = 8;      // query heads of a group served together
constexpr int kWarps = 4;

template <int HD, typename E>
__global__ void __launch_bounds__(32 * kWarps)
    attn_kernel(Kv c, const int32_t* __restrict__ table, int table_ld, int max_pages, const int64_t* __restrict__ pos,
                int H, const E* __restrict__ q, long long q_ld, E* __restrict__ out, long long out_ld,
                float* __restrict__ lse, long long window, float scale) {
  constexpr int PER = HD / 32;
  __shared__ float st[kWarps][GT][HD + 2];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = blockIdx.x, b = blockIdx.z, G = H / c.KV, h0 = g * G + blockIdx.y * GT, nh = min(GT, (g + 1) * G - h0);
  long long hi = pos[b] + 1;
  if (hi < 0) hi = 0;
  const long long room = static_cast<long long>(max_pages) << c.page_shift;
  if (hi > room) {
    if (threadIdx.x == 0) set_status(AIB_DEV_BAD_POS);
    hi = room;
  }
  const long long lo = window > 0 && hi > window ? hi - window : 0;
  float qr[GT][PER], acc[GT][PER], m[GT], l[GT];
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      acc[h][i] = 0.0f;
      float x = 0.0f;
      if (h < nh) load_per<1>(q + b * q_ld + (h0 + h) * HD + lane + 32 * i, 0, &x);
      qr[h][i] = x;
    }
  }
  for (long long j = lo + warp; j < hi; j += kWarps) {
    const int id = table[static_cast<long long>(b) * table_ld + (j >> c.page_shift)];
    if (id < 0 || id >= c.pages) {
      if (lane == 0) set_status(AIB_DEV_BAD_PAGE);
      continue;
    }
    const long long row = id * c.page_stride + g * c.head_stride + (j & ((1 << c.page_shift) - 1)) * c.row_stride;
    float kr[PER], vr[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      kr[i] = bf16_to_f32(c.k[row + lane + 32 * i]);
      vr[i] = bf16_to_f32(c.v[row + lane + 32 * i]);
    }
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) s += qr[h][i] * kr[i];
      s = warp_sum(s) * scale;
      const float mn = fmaxf(m[h], s), al = m[h] == -INFINITY ? 0.0f : expf(m[h] - mn);
      const float p = s == -INFINITY ? 0.0f : expf(s - mn);
      m[h] = mn;
      l[h] = l[h] * al + p;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[h][i] = acc[h][i] * al + p * vr[i];
    }
  }
#pragma unroll
  for (int h = 0; h < GT; ++h) {
#pragma unroll
    for (int i = 0; i < PER; ++i) st[warp][h][lane + 32 * i] = acc[h][i];
    if (lane == 0) {
      st[warp][h][HD] = m[h];
      st[warp][h][HD + 1] = l[h];
    }
  }
  __syncthreads();
  for (int h = 0; h < nh; ++h) {
    float M = -INFINITY, L = 0.0f, wt[kWarps];
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, st[w][h][HD]);
    for (int w = 0; w < kWarps; ++w) {
      wt[w] = st[w][h][HD] == -INFINITY ? 0.0f : expf(st[w][h][HD] - M);
      L += wt[w] * st[w][h][HD + 1];
    }
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
      float a = 0.0f;
      for (int w = 0; w < kWarps; ++w) a += wt[w] * st[w][h][d];
      a = hi > lo && M != -INFINITY ? a / L : 0.0f;
      store_per<1>(out + b * out_ld + (h0 + h) * HD + d, 0, &a);
    }
    if (lse && threadIdx.x == 0) lse[static_cast<long long>(b) * H + h0 + h] = M == -INFINITY ? -INFINITY : M + logf(L);
  }
}

// ----------------------------------------------------------------------------------------- host
static int check_kv(const char* what, const aib_paged_kv* c, Kv* o) {
  if (!c || !c->k || !c->v || c->pages <= 0 || c->KV <= 0) return fail(AIB_EINVAL, "%s: bad cache", what);
  if (c->HD != 64 && c->HD != 128) return fail(AIB_ENOTSUP, "%s: HD must be 64 or 128 (HD=%d)", what, c->HD);
  if (c->page <= 0 || (c->page & (c->page - 1)))
    return fail(AIB_EINVAL, "%s: rows per page must be a power of two (%d)", what, c->page);
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) ||
      ((c->page_stride | c->head_stride | c->row_stride) & 7) || c->page_stride < 0 || c->head_stride < 0 ||
      c->row_stride < 0)
    return fail(AIB_EINVAL, "%s: cache rows must start on 16-byte boundaries, strides must not be negative", what);
  *o = Kv{c->k, c->v, c->page_stride, c->head_stride, c->row_stride, c->pages, c->KV, __builtin_ctz(c->page)};
  return AIB_OK;
}

template <typename E>
static Rows<E> rows_of(const aib_rows* r) {
  if (!r) return Rows<E>{nullptr, 0, 0, 0};
  const bool vec = !(reinterpret_cast<uintptr_t>(r->p) % (2 * sizeof(E))) && !((r->token_stride | r->head_stride) & 1);
  return Rows<E>{static_cast<E*>(r->p), r->token_stride, r->head_stride, vec ? 1 : 0};
}

template <typename E>
static int append(const Kv& c, int HD, const int32_t* table, int table_ld, int max_pages, const int64_t* pos,
                  const int32_t* cu, int B, int T, int H, const aib_rows* q, const aib_rows* k, const aib_rows* v,
                  const aib_rows* qo, const uint16_t* qn, const uint16_t* kn, const float* inv, float eps,
                  cudaStream_t s) {
  const int nv = H + 2 * c.KV;
  const int parts = 1, per = nv;
  const long long warps = static_cast<long long>(T) * parts;
  const dim3 grid(static_cast<unsigned>((warps + kAppWarps - 1) / kAppWarps));
  auto go = [&](auto kernel) {
    return launch(kernel, grid, dim3(32 * kAppWarps), 0, s, "aib_paged_append", c, table, table_ld, max_pages, pos, cu,
                  B, T, H, rows_of<const E>(q), rows_of<const E>(k), rows_of<const E>(v), rows_of<E>(qo), qn, kn, inv,
                  eps, parts, per);
  };
  return HD == 128 ? go(append_kernel<128, E>) : go(append_kernel<64, E>);
}

template <typename E>
static int attend(const Kv& c, int HD, const int32_t* table, int table_ld, int max_pages, const int64_t* pos, int B,
                  int H, const void* q, long long q_ld, void* out, long long out_ld, float* lse, long long window,
                  float scale, cudaStream_t s) {
  const int G = H / c.KV;
  auto go = [&](auto kernel) {
    return launch(kernel, dim3(c.KV, (G + GT - 1) / GT, B), dim3(32 * kWarps), 0, s, "aib_paged_attn", c, table,
                  table_ld, max_pages, pos, H, static_cast<const E*>(q), q_ld, static_cast<E*>(out), out_ld, lse,
                  window, scale);
  };
  return HD == 128 ? go(attn_kernel<128, E>) : go(attn_kernel<64, E>);
}

}  // namespace paged
}  // namespace aib

using namespace aib;

extern "C" {

int aib_paged_append(const aib_paged_kv* cache, const int32_t* table, int table_ld, int max_pages, const int64_t* pos,
                     const int32_t* cu, int B, int T, int H, const aib_rows* q, const aib_rows* k, const aib_rows* v,
                     const aib_rows* q_out, int dtype, const uint16_t* qn, const uint16_t* kn, const float* inv,
                     float eps, void* stream) {
  paged::Kv c;
  const int rc = paged::check_kv("aib_paged_append", cache, &c);
  if (rc) return rc;
  if (!table || !pos || !k || !v || !k->p || !v->p || B <= 0 || T <= 0 || max_pages <= 0 || table_ld < 0 ||
      (dtype != 0 && dtype != 1))
    return fail(AIB_EINVAL, "aib_paged_append: bad arguments");
  if (!cu && T != B) return fail(AIB_EINVAL, "aib_paged_append: without cu, T must be B (T=%d B=%d)", T, B);
  if (H < 0 || (H > 0) != (q && q->p) || (H > 0) != (q_out && q_out->p))
    return fail(AIB_EINVAL, "aib_paged_append: q and q_out go with H > 0");
  if (static_cast<long long>(T) * (H + 2 * c.KV) > 0x7fffffffLL)
    return fail(AIB_ENOTSUP, "aib_paged_append: T * (H + 2 KV) must fit 31 bits");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? paged::append<float>(c, cache->HD, table, table_ld, max_pages, pos, cu, B, T, H, q, k, v, q_out,
                                           qn, kn, inv, eps, s)
                    : paged::append<uint16_t>(c, cache->HD, table, table_ld, max_pages, pos, cu, B, T, H, q, k, v,
                                              q_out, qn, kn, inv, eps, s);
}

size_t aib_paged_attn_workspace(int B, int H, int KV, int HD) {
  if (B <= 0 || H <= 0 || KV <= 0 || H % KV || (HD != 64 && HD != 128)) return 0;
  return 16;
}

int aib_paged_attn(const aib_paged_kv* cache, const int32_t* table, int table_ld, int max_pages, const int64_t* pos,
                   int B, int H, const void* q, int64_t q_ld, void* out, int64_t out_ld, int dtype, float* lse,
                   int64_t window, float scale, void* ws, size_t ws_bytes, void* stream) {
  paged::Kv c;
  const int rc = paged::check_kv("aib_paged_attn", cache, &c);
  if (rc) return rc;
  if (!table || !pos || !q || !out || B <= 0 || B > 65535 || max_pages <= 0 || table_ld < 0 || window < 0 ||
      (dtype != 0 && dtype != 1) || H <= 0 || H % c.KV || q_ld < 0 || out_ld < 0)
    return fail(AIB_EINVAL, "aib_paged_attn: bad arguments");
  if (!ws || ws_bytes < aib_paged_attn_workspace(B, H, c.KV, cache->HD))
    return fail(AIB_EWORKSPACE, "aib_paged_attn: workspace %zu < %zu bytes", ws_bytes,
                aib_paged_attn_workspace(B, H, c.KV, cache->HD));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? paged::attend<float>(c, cache->HD, table, table_ld, max_pages, pos, B, H, q, q_ld, out, out_ld,
                                           lse, window, scale, s)
                    : paged::attend<uint16_t>(c, cache->HD, table, table_ld, max_pages, pos, B, H, q, q_ld, out,
                                              out_ld, lse, window, scale, s);
}

}  // extern "C"
