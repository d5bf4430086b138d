// Paged key-value cache (sm_100a): appending new tokens with q/k norm and position rotation, and attention of one new
// token per sequence. No counterpart in the reference, whose caches are contiguous (core/engine.py:234-235); the
// arithmetic is that of qk_rope_cache_k and attn_k (kernels/tkernels.py:82-150).
//
// Sequence b's row at position p is row p % page of page table[b * table_ld + p / page] of the pool. Device data is
// checked where it is used: a position past the table's last page records AIB_DEV_BAD_POS, a page id outside the pool
// AIB_DEV_BAD_PAGE, and the row is neither written nor attended.
#include <algorithm>
#include <atomic>
#include <cfloat>
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
// [T, heads, HD] rows: token and head strides in elements, inner stride 1
template <typename E>
struct Rows {
  E* p;
  long long ts, hs;
};

// Four neighbouring elements as floats and back; VEC: in one access (16 bytes of fp32, 8 of bf16), evicted first since they
// are read once (16384 prompt tokens: 135 us with plain loads, 119 us with these).
template <bool VEC>
AIB_DEV void load4(const float* p, float* o) {
  if (VEC) {
    const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
    o[0] = t.x, o[1] = t.y, o[2] = t.z, o[3] = t.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = p[i];
  }
}
template <bool VEC>
AIB_DEV void load4(const uint16_t* p, float* o) {
  if (VEC) {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
    o[0] = __uint_as_float(t.x << 16), o[1] = __uint_as_float(t.x & 0xFFFF0000u);
    o[2] = __uint_as_float(t.y << 16), o[3] = __uint_as_float(t.y & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = bf16_to_f32(p[i]);
  }
}
AIB_DEV void store4(float* p, float4 a, bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = a;
  } else {
    p[0] = a.x, p[1] = a.y, p[2] = a.z, p[3] = a.w;
  }
}
AIB_DEV void store4(uint16_t* p, float4 a, bool vec) {
  const uint32_t lo = bf16x2_rn(a.x, a.y), hi = bf16x2_rn(a.z, a.w);
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
  } else {
    p[0] = lo & 0xFFFF, p[1] = lo >> 16, p[2] = hi & 0xFFFF, p[3] = hi >> 16;
  }
}
AIB_DEV float to_f32(float x) { return x; }
AIB_DEV float to_f32(uint16_t x) { return bf16_to_f32(x); }
AIB_DEV void from_f32(float x, float* o) { *o = x; }
AIB_DEV void from_f32(float x, uint16_t* o) { *o = bf16_rn(x); }

// cos and sin of p * inv. The product is formed in 64 bits (exact: 31 x 24 bits fit with at most one rounding in the
// last place) and reduced by whole turns there, so a far position loses nothing; a float product would be off by
// p * 2^-24 radians.
AIB_DEV void rotation(long long p, float inv, float* c, float* s) {
  const double a = static_cast<double>(p) * static_cast<double>(inv);
  const double n = rint(a * 0.15915494309189533577);
  const float r = static_cast<float>(fma(-n, 6.283185307179586477, a));
  sincosf(r, s, c);
}

// The sequence of token t (cu NULL: one token each) and its position: b, the position's first token's, the offset.
// Sequences are found 32 places a round, with the positions of the places probed read along with them. cu is device
// data: whatever it holds, b is in range. False for a row behind the last sequence.
AIB_DEV bool find_seq(const int32_t* cu, const int64_t* pos, int B, int t, int* b, long long* p0, int* off) {
  if (!cu) {
    *b = t;
    *p0 = pos[t];
    *off = 0;
    return true;
  }
  const int lane = threadIdx.x & 31, total = cu[B];
  int lo = 0, hi = B, c = 0;
  long long p = 0;
  while (true) {
    const int step = (hi - lo + 31) / 32, i = lo + lane * step;
    if (i < hi) {
      c = cu[i];
      p = pos[i];
    }
    const int n = max(1, __popc(__ballot_sync(0xffffffffu, i < hi && c <= t)));
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
    if (step == 1 || hi - lo == 1) {
      *b = lo;
      *off = t - __shfl_sync(0xffffffffu, c, n - 1);
      *p0 = __shfl_sync(0xffffffffu, p, n - 1);
      return t < total && *off >= 0;
    }
  }
}

// One warp takes `per` of a token's head vectors (q heads, then k heads, then v heads), several at a time: a vector has
// LPV lanes, a lane four dimensions from r on and their rotation partners HD/2 further, so a vector is read and written
// with 16-byte accesses and norm and rotation need no exchange but the sum of squares. The norm's weights are folded
// into the token's cosines and sines, which a warp computes once. The first vectors are on their way before the warp
// looks for its sequence, position and page, the next ones while it works.
// Bound by bytes for prompts: 16384 tokens of 32 + 2 x 8 heads of 128 in fp32, 738 MB, 118 us = 6.25 TB/s captured (two
// dimensions a lane and norm weights read for every vector: 131 instructions a vector and 135 us). By latency for single
// tokens: 2.4 us among captured calls, 4.2 us by itself (18 us when one warp did all of its 48 vectors).
constexpr int kAppWarps = 8;
constexpr int kAppSteps = 2;  // steps of 32 / LPV vectors in hand, and as many on their way

template <int HD, typename E, bool VEC>
__global__ void __launch_bounds__(32 * kAppWarps)
    append_kernel(Kv c, const int32_t* __restrict__ table, long long table_ld, int max_pages,
                  const int64_t* __restrict__ pos, const int32_t* __restrict__ cu, int B, int T, int H, Rows<const E> q,
                  Rows<const E> k, Rows<const E> v, Rows<E> qo, const uint16_t* __restrict__ qn,
                  const uint16_t* __restrict__ kn, const float* __restrict__ inv, float eps, int parts, int per) {
  constexpr int LPV = HD / 8, VPW = 32 / LPV, HALF = HD / 2, BATCH = kAppSteps * VPW;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, sub = lane / LPV, r = lane % LPV * 4;
  const unsigned w = blockIdx.x * kAppWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(w / parts);
  if (t >= T) return;
  const int KV = c.KV, nv = H + 2 * KV, v0 = static_cast<int>(w % parts) * per, v1 = min(nv, v0 + per);
  // a batch has vectors of one kind: [h0, stop)
  auto stop_of = [&](int h0) { return min(min(h0 + BATCH, v1), h0 < H ? H : (h0 < H + KV ? H + KV : nv)); };
  auto load = [&](int h0, float (*x)[8]) {
    if (h0 >= v1) return;
    const Rows<const E> src = h0 < H ? q : (h0 < H + KV ? k : v);
    const int first = h0 < H ? 0 : (h0 < H + KV ? H : H + KV), stop = stop_of(h0);
    const E* p = src.p + t * src.ts + (h0 - first + sub) * src.hs + r;
#pragma unroll
    for (int i = 0; i < kAppSteps; ++i) {
      if (h0 + sub + i * VPW < stop) {
        load4<VEC>(p, x[i]);
        load4<VEC>(p + HALF, x[i] + 4);
      }
      p += VPW * src.hs;
    }
  };
  float x[kAppSteps][8];
  load(v0, x);
  float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (inv) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = inv[r + i];
  }
  int b, off;
  long long p0;
  if (!find_seq(cu, pos, B, t, &b, &p0, &off) || p0 < 0) return;  // behind the last sequence, or an unused row
  // A position near 2^63 wraps below zero behind its offset: past every table, like the position itself.
  const long long p = static_cast<long long>(static_cast<unsigned long long>(p0) + static_cast<unsigned>(off));
  // where the token's k and v rows go
  long long row = -1;
  if (v1 > H) {
    const long long pg = p >> c.page_shift;
    if (p < 0 || pg >= max_pages) {
      if (lane == 0) set_status(AIB_DEV_BAD_POS);
    } else {
      const int id = table[b * table_ld + pg];
      if (id < 0 || id >= c.pages) {
        if (lane == 0) set_status(AIB_DEV_BAD_PAGE);
      } else {
        row = id * c.page_stride + (p & ((1 << c.page_shift) - 1)) * c.row_stride;
      }
    }
  }
  float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (inv && v0 < H + KV) {  // the warp's groups share the four angles
    constexpr int PER = 4 / VPW;
    float ca[PER], sa[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float mine = f[i];
#pragma unroll
      for (int s = 1; s < VPW; ++s) mine = sub == s ? f[s * PER + i] : mine;
      rotation(p, mine, &ca[i], &sa[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = __shfl_sync(0xffffffffu, ca[i % PER], i / PER * LPV + lane % LPV);
      sn[i] = __shfl_sync(0xffffffffu, sa[i % PER], i / PER * LPV + lane % LPV);
    }
  }
  float ac[4], as[4], zc[4], zs[4];  // weight times cosine or sine, of the first half's and of the second's elements
  int kind = -1;
  for (int h0 = v0; h0 < v1;) {
    const int stop = stop_of(h0), now = h0 < H ? 0 : (h0 < H + KV ? 1 : 2);
    float y[kAppSteps][8];
    load(stop, y);
    const uint16_t* wn = now == 0 ? qn : kn;
    if (now != kind && now != 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float wa = wn ? bf16_to_f32(wn[r + j]) : 1.0f, wz = wn ? bf16_to_f32(wn[r + j + HALF]) : 1.0f;
        ac[j] = wa * cs[j];
        as[j] = wa * sn[j];
        zc[j] = wz * cs[j];
        zs[j] = wz * sn[j];
      }
    }
    kind = now;
#pragma unroll
    for (int i = 0; i < kAppSteps; ++i) {
      const int h = h0 + sub + i * VPW;
      const bool mine = h < stop;
      float4 lo = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]), hi = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
      if (now != 2) {
        float rs = 1.0f;
        if (wn) {
          float ss = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += x[i][j] * x[i][j];
#pragma unroll
          for (int o = LPV / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          rs = rsqrtf(ss * (1.0f / HD) + eps);
        }
        float a[4], z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // without rotation nothing of the partner enters (0 times an infinity would)
          a[j] = rs * (inv ? x[i][j] * ac[j] - x[i][4 + j] * zs[j] : x[i][j] * ac[j]);
          z[j] = rs * (inv ? x[i][4 + j] * zc[j] + x[i][j] * as[j] : x[i][4 + j] * zc[j]);
        }
        lo = make_float4(a[0], a[1], a[2], a[3]);
        hi = make_float4(z[0], z[1], z[2], z[3]);
      }
      if (!mine) continue;
      if (now == 0) {
        E* dst = qo.p + t * qo.ts + h * qo.hs + r;
        store4(dst, lo, VEC);
        store4(dst + HALF, hi, VEC);
      } else if (row >= 0) {
        uint16_t* dst = now == 1 ? c.k + row + (h - H) * c.head_stride + r : c.v + row + (h - H - KV) * c.head_stride + r;
        store4(dst, lo, true);
        store4(dst + HALF, hi, true);
      }
    }
#pragma unroll
    for (int i = 0; i < kAppSteps; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = y[i][j];
    h0 = stop;
  }
}

// ---------------------------------------------------------------------------------- attention
// out = sum_j softmax_j(scale q.k_j) v_j in one pass over the rows with a running maximum and sum (in base 2).
//
// Split: the work is a line of units, a unit being 32 cached rows (from a multiple of 32) of one (sequence, key head,
// tile of 8 query heads). Every CTA, one an SM, takes an equal run of the line and every warp an equal piece of the run,
// so the load does not depend on how ragged the lengths are and the host need not know them (a captured step keeps its
// grid while the sequences grow). A (sequence, head) that lies inside one warp's piece is finished there, so short
// sequences need no joining; where it crosses warps their states are joined in shared memory at the end of the run;
// where it crosses CTAs each writes a partial state and the last one to finish (a ticket; nobody waits) joins them. All
// joins run in the order of the line, so the sums do not depend on timing.
//
// A warp copies for itself: its lanes look up the pages of its next 32 boxes at once (a box: the rows of a page, 32 at
// most), and one tensor copy brings a box of K or V into one of the warp's three tiles of shared memory, K of unit i + 2
// as soon as V of unit i is used up, V of unit i + 1 when K of unit i is. The copies land in the 128-byte swizzle, so the
// eight row addresses of an ldmatrix hit different banks. No warp waits for another before the end of its run.
//
// Masked rows (outside the span, or on a page outside the pool) get weight 0 and their V rows are cleared in shared
// memory, whatever the cache holds there; boxes without a row to attend are not fetched.
//
// The few query rows (at most 8 a tile) go through mma.sync as the 8 columns: the kernel is bound by the cache's bytes,
// and the tensor cores are far from their limit (3 products of 16 x 8 x 16 a 16 x 16 piece of K or V). fp32 rows enter as
// three bf16 parts and so do their weights (24 bits, as good as fp32 products); bf16 rows are exact as they are, and
// their weights take two parts (16 bits, 2^-8 of the output's own rounding). An mma chops its sums where an fp32 addition
// rounds, so no long chain runs through one accumulator: the rows' running sums are added outside (131072 rows in fp32:
// error 3.9e-6 with one accumulator, 3.6e-7 so).
//
// Measured (B200, captured, caches in turn so that none is left in L2): 64 sequences of up to 8192 in bf16, 983 MB, 157 us =
// 6.3 TB/s; one of 131072 in fp32, 537 MB, 93 us = 5.8 TB/s (a few SMs get 12 % less of the memory and finish last); 16 of up
// to 4096 32 us, of which about 21 us are the copies, the rest the sum over the lengths, the first look-up and the joins; 200
// windowed ones 26 us; one of 517 11 us, all latency. Query heads beyond 8 a key head are another tile, which reads the same
// rows again (16 sequences of up to 8192, 8 x 16 heads of 128, bf16: 82 us cold, twice its floor of 41).
// Tried and slower: a copying warp for eight computing ones (single units, 190 us for the 64 sequences: it issued too
// slowly; batches of look-ups, 157 us, but 36 against 25 us for 200 short ones, whose joins held the warps up), 16-byte
// asynchronous copies (178 us), runs of two sizes (no change), the joins' code run once ahead of time (+5 us).
constexpr int GT = 8;       // query heads of a group served together (the columns of an mma)
constexpr int kBlk = 32;    // rows of a unit
constexpr int kTiles = 3;   // tiles of a warp
constexpr int kMaxBatch = 4096;
constexpr int kMaxGrid = 256;

template <int HD>
struct Lay {
  static constexpr int kWarps = HD == 128 ? 8 : 12;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kTile = kBlk * HD * 2;           // the K or V rows of a unit: its boxes one after the other
  static constexpr int kRing = kWarps * kTiles * kTile;
  static constexpr int kW = HD + 4;                     // a head's sums, its maximum, its sum of weights, padding
  static constexpr int kPart = GT * kW;                 // floats of a state
  static constexpr int kMinRun = 8;                     // units of a CTA's run at least
  static_assert(kTiles * kTile >= kPart * 4, "a warp's last state goes where its tiles were");
  static_assert(2 * kWarps <= 32, "a lane for every state");
};

// Rows [row, row + box) of head kvh in page id: [HD / 64][box][64] elements in shared memory, 128-byte swizzle.
template <int HD>
AIB_DEV void tma_load(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int row, int kvh, int id, uint64_t policy) {
  if (HD == 128)
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, "
        "%3, %5, %6}], [%2], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(kvh), "r"(id), "l"(policy)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, "
        "%5, %6}], [%2], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(kvh), "r"(id), "l"(policy)
        : "memory");
}
template <int N>
AIB_DEV void split_pair(float lo, float hi, uint32_t* w) {  // lo, hi as N bf16 parts each, (hi << 16) | lo
#pragma unroll
  for (int k = 0; k < N; ++k) {
    w[k] = bf16x2_rn(lo, hi);
    lo -= __uint_as_float(w[k] << 16);
    hi -= __uint_as_float(w[k] & 0xFFFF0000u);
  }
}
// Two fp32 numbers as three bf16 parts, exactly: 8 bits of the 24 each, cut off and not rounded, so that a number above the
// largest bf16 one does not round to infinity. An infinity leaves NaN behind. N 1: numbers that are bf16 already.
template <int N>
AIB_DEV void split_exact(float lo, float hi, uint32_t* w) {
  static_assert(N == 1 || N == 3, "24 bits in parts of 8, or 8");
#pragma unroll
  for (int k = 0; k < N; ++k) {
    w[k] = prmt(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
    lo -= __uint_as_float(__float_as_uint(lo) & 0xFFFF0000u);
    hi -= __uint_as_float(__float_as_uint(hi) & 0xFFFF0000u);
  }
}
AIB_DEV uint32_t transpose8(uint32_t x) {  // an 8 x 8 matrix of 16-bit elements, a row to four lanes
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Rows [lo, hi) that sequence b attends; false if its position lies past the table.
AIB_DEV bool span(const int64_t* pos, int b, int room, long long window, int* lo, int* hi) {
  const long long p = pos[b];
  const bool ok = p < room;
  *hi = p < 0 ? 0 : (ok ? static_cast<int>(p) + 1 : room);
  *lo = 0;
  if (window > 0 && p >= window) *lo = static_cast<int>(min(p - window + 1, static_cast<long long>(*hi)));
  return ok;
}
AIB_DEV int units_of(int lo, int hi) { return hi > lo ? (hi - 1) / kBlk - lo / kBlk + 1 : 0; }

// A place in a CTA's run: sequence b, its part (a tile of a key head's query heads), whose units are [seg0, seg0 + nblk),
// counted from the run's first unit (seg0 is negative where the part began in an earlier run).
struct Cursor {
  int seg0, nblk, b, kvh, tile, lo, hi;
};
struct Line {
  const int64_t* pos;
  long long window;
  int B, room, KV, tiles;
};
AIB_DEV void enter(Cursor& c, const Line& l) {
  span(l.pos, c.b, l.room, l.window, &c.lo, &c.hi);
  c.nblk = units_of(c.lo, c.hi);
}
AIB_DEV void seek(Cursor& c, const Line& l, int u) {  // forward to the part that holds unit u
  while (u - c.seg0 >= c.nblk) {
    c.seg0 += c.nblk;
    if (++c.tile == l.tiles) {
      c.tile = 0;
      ++c.kvh;
    }
    if (c.kvh == l.KV) {
      c.kvh = 0;
      do {
        if (++c.b >= l.B) {  // not reached while pos stays as it was
          c.b = l.B - 1;
          c.nblk = 0x7fffffff;
          c.lo = c.hi = 0;
          return;
        }
        enter(c, l);
      } while (c.nblk == 0);
    }
  }
}

AIB_DEV void add4(float4& a, float w, float4 x) {
  a.x += w * x.x;
  a.y += w * x.y;
  a.z += w * x.z;
  a.w += w * x.w;
}
// No row attended: no maximum and no weights.
AIB_DEV bool nothing(float M, float L) { return M == -INFINITY && L == 0.0f; }
AIB_DEV float lse_of(float M, float L) {
  return nothing(M, L) ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}
// Four neighbouring outputs (from dimension d) of a head from its sums.
template <typename E>
AIB_DEV void write_out(E* out, float* lse, float M, float L, float4 a, int d, bool vec) {
  const float r = 1.0f / L;
  store4(out + d, nothing(M, L) ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(a.x * r, a.y * r, a.z * r, a.w * r),
         vec);
  if (lse && d == 0) *lse = lse_of(M, L);
}

// Adds 1 and returns what was there: everything this CTA wrote before its last barrier is visible to who reads after a
// later ticket.
AIB_DEV int ticket(int* p) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}

struct Owner {  // what a state in shared memory belongs to: heads h0 .. h0 + nh - 1 of b (b < 0: there is none)
  int b, h0, nh, seg0, nblk;
};
// a / b for a that is nearly always below 2^31 (a 64-bit division takes most of a microsecond)
AIB_DEV long long quotient(long long a, int b) {
  return a >> 31 ? a / b : static_cast<unsigned>(a) / static_cast<unsigned>(b);
}
template <int HD>
struct Shared {
  uint64_t full[Lay<HD>::kWarps][kTiles];
  long long wtot[Lay<HD>::kWarps], base;
  Owner own[2 * Lay<HD>::kWarps];  // the warps' first states (parts that began before the piece) and last states
  int b, abort, last[2], c0[2], np[2];
};

template <int HD, typename E>
__global__ void __launch_bounds__(Lay<HD>::kThreads, 1)
    attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int pages, int KV,
                int page_shift, const int32_t* __restrict__ table, long long table_ld, int room,
                const int64_t* __restrict__ pos, int B, int H, const E* __restrict__ q, long long q_ld,
                E* __restrict__ out, long long out_ld, float* __restrict__ lse, long long window, float scale, int* cnt,
                float* parts_ws) {
  using Y = Lay<HD>;
  constexpr int PQ = sizeof(E) == 4 ? 3 : 1, PP = sizeof(E) == 4 ? 3 : 2;
  constexpr int NT = HD / 16, W = Y::kW, NW = Y::kWarps;
  extern __shared__ uint8_t dyn[];
  uint8_t* ring = dyn + (-smem_u32(dyn) & 1023u);
  float* first = reinterpret_cast<float*>(ring + Y::kRing);
  Shared<HD>& sh = *reinterpret_cast<Shared<HD>*>(first + NW * Y::kPart);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, grid = gridDim.x;
  const int G = H / KV, tiles = (G + GT - 1) / GT;
  const Line line{pos, window, B, room, KV, tiles};
  const int parts = KV * tiles;
  if (lane < kTiles) mbar_init(&sh.full[warp][lane], 1);
  if (lane < 2) sh.own[2 * warp + lane].b = -1;
  if (threadIdx.x == 0) {
    sh.abort = 0;
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  fence_mbar_init();
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's run, n units from u0: a sum over the sequences' units, every thread over a few of them
  const int cb = (B + Y::kThreads - 1) / Y::kThreads, b_lo = min(B, static_cast<int>(threadIdx.x) * cb),
            b_hi = min(B, b_lo + cb);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    int lo, hi;
    if (!span(pos, b, room, window, &lo, &hi) && cta == 0) set_status(AIB_DEV_BAD_POS);
    mine += units_of(lo, hi);
  }
  mine *= parts;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.wtot[warp] = incl;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += sh.wtot[w];
    total += sh.wtot[w];
  }
  const int per = static_cast<int>(max(static_cast<long long>(Y::kMinRun), quotient(total + grid - 1, grid)));
  const long long u0 = static_cast<long long>(cta) * per;
  const int n = static_cast<int>(max(0LL, min(total - u0, static_cast<long long>(per))));
  if (n > 0) {
    long long base = before + incl - mine;
    if (u0 >= base && u0 < base + mine) {
      for (int b = b_lo; b < b_hi; ++b) {
        int lo, hi;
        span(pos, b, room, window, &lo, &hi);
        const long long m = static_cast<long long>(units_of(lo, hi)) * parts;
        if (u0 < base + m) {
          sh.b = b;
          sh.base = base;
          break;
        }
        base += m;
      }
    }
  }
  __syncthreads();

  // ---- the warp's piece [beg, end) of the run
  const int piece = (n + NW - 1) / NW, beg = min(n, warp * piece), end = min(n, beg + piece);
  const bool vec = !((reinterpret_cast<uintptr_t>(out) | out_ld * sizeof(E)) % (4 * sizeof(E)));
  if (beg < end) {
    Cursor C;
    C.b = sh.b;
    enter(C, line);
    const int part = static_cast<int>(quotient(u0 - sh.base, C.nblk));
    C.seg0 = -static_cast<int>(u0 - sh.base - static_cast<long long>(part) * C.nblk);
    C.kvh = part / tiles;
    C.tile = part - C.kvh * tiles;
    seek(C, line, beg);

    // copies: a lane stands for a box of a unit
    Cursor P = C;
    const int box = min(kBlk, 1 << page_shift), nbox = kBlk / box, batch = 32 / nbox;  // units of a batch
    const int bx = lane & (nbox - 1), bu = lane / nbox;                                // the lane's box, its unit
    struct Look {
      int id, row, kvh;
      uint32_t rows;  // the box's rows that are attended, as bits of the unit
    };
    auto look_up = [&](int u) {
      Look k{-1, 0, 0, 0};
      if (u + bu < end) {
        seek(P, line, u + bu);
        const int j0 = (P.lo & ~(kBlk - 1)) + (u + bu - P.seg0) * kBlk, a = j0 + bx * box;
        const int r0 = max(a, P.lo) - j0, r1 = min(a + box, P.hi) - j0;  // within the unit
        k.kvh = P.kvh;
        k.row = a & ((1 << page_shift) - 1);
        if (r0 < r1) {
          k.rows = (0xffffffffu >> (32 - (r1 - r0))) << r0;
          k.id = table[P.b * table_ld + (a >> page_shift)];
        }
      }
      return k;
    };
    uint8_t* my_ring = ring + warp * kTiles * Y::kTile;
    const uint32_t tile0 = smem_u32(my_ring);
    Look now{-1, 0, 0, 0}, next = look_up(beg);
    uint32_t mask = 0, bytes = 0;       // of the lane's unit
    int at = batch, iu = beg, is = 0;   // place in the batch of the unit whose copies start next, that unit, its tile
    int started = 0, landed = 0;        // copies of the warp
    const bool withhold = g_aib_withhold_copies != 0;
    // With one tile of query heads a call reads the cache once, so its copies leave L2 first. In a step other data pass between
    // two visits of a layer's cache; caches in turn, 600 MB of them: 16 sequences of up to 4096 32.2 us, 200 windowed ones 26.8
    // (without the hint 33.4 and 28.9; a cache that is all in L2 loses, 26.0 and 24.3 us for the windowed one over and over).
    // With several tiles every one reads the same rows again, and the copies stay as others do: 16 query heads to a key head,
    // bf16, L2 cold, 16 sequences: 8 key heads, up to 8192 rows 84 us (evicted first 96), one, up to 32768 rows 47 us (55).
    const uint64_t policy = tiles == 1 ? l2_evict_first() : l2_evict_normal();
    // starts the copies of unit iu's K (and returns the unit's attended rows) or V
    auto start = [&](bool v) {
      if (!v && at == batch) {
        at = 0;
        now = next;
        if (now.rows && (now.id < 0 || now.id >= pages)) {
          set_status(AIB_DEV_BAD_PAGE);
          now.rows = 0;
        }
        mask = now.rows;
        bytes = now.rows ? box * HD * 2 : 0;
        for (int o = 1; o < nbox; o <<= 1) {
          mask |= __shfl_xor_sync(0xffffffffu, mask, o);
          bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
        }
        next = look_up(iu + batch);
      }
      uint64_t* bar = &sh.full[warp][is];
      if (withhold) return 0u;  // test knob 2: the tile never fills
      if (lane == at * nbox) mbar_arrive_expect_tx(bar, bytes);
      __syncwarp();
      if (bu == at && now.rows)
        tma_load<HD>(tile0 + is * Y::kTile + bx * box * HD * 2, v ? &vmap : &kmap, bar, now.row, now.kvh, now.id, policy);
      const uint32_t vm = __shfl_sync(0xffffffffu, mask, at * nbox);
      ++started;
      is = is == kTiles - 1 ? 0 : is + 1;
      if (v) {
        ++at;
        ++iu;
      }
      return vm;
    };
    uint32_t vm = start(false), vm_next = 0;
    start(true);
    if (iu < end) vm_next = start(false);

    // ldmatrix rows: box by box, [HD / 64][box][128 bytes]. The 16-byte chunk c of the 128 bytes at address a lies in
    // chunk c ^ (a / 128 % 8): `place` gives a with that number in the chunk's bits, to be combined with c by one xor.
    const int box_shift = min(5, page_shift);
    auto place = [&](int row, int half) {
      const uint32_t a =
          ((row >> box_shift << box_shift) * (HD / 64) + (half << box_shift) + (row & ((1 << box_shift) - 1))) * 128;
      return a | ((a >> 7 & 7) << 4);
    };
    const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kcol = lane >> 4;  // A tile of K rows: row, chunk
    const int vr = (lane & 7) + (lane >> 4) * 8, vcol = (lane >> 3) & 1;  // V tile, transposed load
    uint32_t ka[2][HD / 64], va[2][HD / 64];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < HD / 64; ++h) {
        ka[m][h] = place(m * 16 + kr, h) ^ kcol << 4;
        va[m][h] = place(m * 16 + vr, h) ^ vcol << 4;
      }
    const float sl = scale * 1.4426950408889634f;
    int cs = 0, ph = 0, u = beg;  // tile and parity of the next wait
    bool ok = true;
    auto wait = [&]() {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&sh.full[warp][cs], ph, AIB_DEV_TIMEOUT_FULL));
      const int tile = cs;
      if (ok) ++landed;
      if (++cs == kTiles) {
        cs = 0;
        ph ^= 1;
      }
      return tile;
    };
    while (true) {
      const int h0 = C.kvh * G + C.tile * GT, nh = min(GT, G - C.tile * GT);
      const int stop = min(end, C.seg0 + C.nblk);
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
      float acc[NT][4];
#pragma unroll
      for (int d = 0; d < NT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.0f;
      uint32_t bq[NT][PQ][2];  // q of head g, dimensions 16 s + 2t, +1 and +8, +9
      const E* qr = q + C.b * q_ld + static_cast<long long>(h0 + min(g, nh - 1)) * HD + 2 * t;
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        const float x[4] = {to_f32(qr[16 * s]), to_f32(qr[16 * s + 1]), to_f32(qr[16 * s + 8]), to_f32(qr[16 * s + 9])};
        uint32_t w0[PQ], w1[PQ];
        split_exact<PQ>(x[0], x[1], w0);
        split_exact<PQ>(x[2], x[3], w1);
#pragma unroll
        for (int k = 0; k < PQ; ++k) bq[s][k][0] = w0[k], bq[s][k][1] = w1[k];
      }
      for (; u < stop; ++u) {
        const uint32_t kt = tile0 + wait() * Y::kTile;
        if (!ok) break;
        float sc[2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          // the leading parts' products in two chains, the small parts' in a third
          float x[3][4] = {};
#pragma unroll
          for (int s = 0; s < NT; ++s) {
            uint32_t a0, a1, a2, a3;
            attn::ldsm_x4(kt + (ka[mt][s / 4] ^ (s % 4 * 32)), a0, a1, a2, a3);
            mma_bf16(x[s & 1], a0, a1, a2, a3, bq[s][0][0], bq[s][0][1]);
#pragma unroll
            for (int k = 1; k < PQ; ++k) mma_bf16(x[2], a0, a1, a2, a3, bq[s][k][0], bq[s][k][1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[mt][i] = x[0][i] + x[1][i] + x[2][i];
        }
        __syncwarp();
        if (iu < end) start(true);  // V of the next unit goes where this one's K was
        // weights: sc[mt][0/1] are heads 2t, 2t+1 at row mt*16 + g, sc[mt][2/3] at row mt*16 + g + 8
        float s0[4], s1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = vm >> ((i >> 1) * 16 + g + (i & 1) * 8) & 1;
          s0[i] = in ? sc[i >> 1][(i & 1) * 2] * sl : -INFINITY;
          s1[i] = in ? sc[i >> 1][(i & 1) * 2 + 1] * sl : -INFINITY;
        }
        float b0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3])), b1 = fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, o));
          b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, o));
        }
        // With a row to attend the maximum is finite at least, so that a head whose scores are all -inf (sum 0, NaN by the
        // definition) can be told from one that attends nothing.
        const float least = vm ? -FLT_MAX : -INFINITY;
        const float n0 = fmaxf(fmaxf(m0, b0), least), n1 = fmaxf(fmaxf(m1, b1), least);
        const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;  // no row so far: weights 0
        const float al0 = exp2f(m0 - z0), al1 = exp2f(m1 - z1);
        m0 = n0;
        m1 = n1;
        l0 *= al0;
        l1 *= al1;
        // the weights' parts, turned from (row g, heads 2t, 2t+1) to (head g, rows 2t, 2t+1) eight rows at a time. Every
        // lane keeps the sum over its own rows; the lanes' sums are added at the end of the part.
        uint32_t bp[4][PP];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = exp2f(s0[i] - z0), p1 = exp2f(s1[i] - z1);
          l0 += p0;
          l1 += p1;
          split_pair<PP>(p0, p1, bp[i]);
#pragma unroll
          for (int k = 0; k < PP; ++k) bp[i][k] = transpose8(bp[i][k]);
        }
        const int v_tile = wait();
        if (!ok) break;
        const uint32_t vt = tile0 + v_tile * Y::kTile;
        if (vm != 0xffffffffu) {  // clear the V rows that are not attended (the tile's next copy comes after this)
          if (!(vm >> lane & 1)) {
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
              uint4* row = reinterpret_cast<uint4*>(my_ring + v_tile * Y::kTile + (place(lane, h) & ~127u));
#pragma unroll
              for (int c = 0; c < 8; ++c) row[c] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async();
          __syncwarp();
        }
#pragma unroll
        for (int d = 0; d < NT; ++d) {
          float x[4] = {};
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            uint32_t a0, a1, a2, a3;
            attn::ldsm_x4_t(vt + (va[s][d / 4] ^ (d % 4 * 32)), a0, a1, a2, a3);
#pragma unroll
            for (int k = PP - 1; k >= 0; --k) mma_bf16(x, a0, a1, a2, a3, bp[2 * s][k], bp[2 * s + 1][k]);
          }
          acc[d][0] = acc[d][0] * al0 + x[0];
          acc[d][1] = acc[d][1] * al1 + x[1];
          acc[d][2] = acc[d][2] * al0 + x[2];
          acc[d][3] = acc[d][3] * al1 + x[3];
        }
        __syncwarp();
        vm = vm_next;
        if (iu < end) vm_next = start(false);  // K of the unit after the next goes where this one's V was
      }
      if (!ok) break;
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
      }
      const bool began = C.seg0 >= beg, ended = C.seg0 + C.nblk <= end;
      if (began && ended) {
        E* o = out + C.b * out_ld + static_cast<long long>(h0) * HD + g;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int h = 2 * t + hh;
          const float M = hh ? m1 : m0, L = hh ? l1 : l0, r = 1.0f / L;
          const bool none = nothing(M, L);
          if (h < nh) {
#pragma unroll
            for (int d = 0; d < NT; ++d) {
              const float x = none ? 0.0f : acc[d][hh] * r, y = none ? 0.0f : acc[d][2 + hh] * r;
              from_f32(x, o + h * HD + d * 16);
              from_f32(y, o + h * HD + d * 16 + 8);
            }
            if (lse && g == 0) lse[static_cast<long long>(C.b) * H + h0 + h] = lse_of(M, L);
          }
        }
      } else {
        float* st = ended ? first + warp * Y::kPart : reinterpret_cast<float*>(my_ring);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float* dst = st + (2 * t + hh) * W;
#pragma unroll
          for (int d = 0; d < NT; ++d) {
            dst[d * 16 + g] = acc[d][hh];
            dst[d * 16 + g + 8] = acc[d][2 + hh];
          }
          if (g == 0) {
            dst[HD] = hh ? m1 : m0;
            dst[HD + 1] = hh ? l1 : l0;
          }
        }
        if (lane == 0) sh.own[2 * warp + (ended ? 0 : 1)] = Owner{C.b, h0, nh, C.seg0, C.nblk};
      }
      if (u >= end) break;
      seek(C, line, u);
    }
    if (!ok) {  // a wait ran out: the copies that are still on their way must land before the CTA ends
      sh.abort = 1;
      for (int k = landed; k < started; ++k)
        for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(&sh.full[warp][k % kTiles], k / kTiles & 1); ++i) {
        }
    }
  }
  __syncthreads();

  // ---- parts that cross warps: their states, neighbours among the 2 NW places, are joined in order
  Owner o{-1, 0, 0, 0, 0};
  if (lane < 2 * NW) o = sh.own[lane];
  const uint32_t there = sh.abort ? 0 : __ballot_sync(0xffffffffu, o.b >= 0);
  if (there) {
    const uint32_t below = there & ((1u << lane) - 1);
    const int prev = below ? 31 - __clz(below) : 0;
    const int pb = __shfl_sync(0xffffffffu, o.b, prev), ph0 = __shfl_sync(0xffffffffu, o.h0, prev);
    const uint32_t heads = __ballot_sync(0xffffffffu, o.b >= 0 && (!below || pb != o.b || ph0 != o.h0));
    // items of four dimensions: as many heads a group as the next power of two, HD / 4 items a head
    const int ng = __popc(heads), head_bits = 32 - __clz(min(G, GT) - 1);
    constexpr int kItemBits = HD == 128 ? 5 : 4;
    for (int i = threadIdx.x; i < ng << (head_bits + kItemBits); i += Y::kThreads) {
      uint32_t rest = heads;
      for (int k = i >> (head_bits + kItemBits); k > 0; --k) rest &= rest - 1;
      const int lo = __ffs(rest) - 1;
      rest &= rest - 1;
      const uint32_t set = there & (0xffffffffu << lo) & (rest ? (1u << (__ffs(rest) - 1)) - 1 : 0xffffffffu);
      const Owner w = sh.own[lo];
      const int h = i >> kItemBits & ((1 << head_bits) - 1), d = i % (HD / 4) * 4;
      if (h >= w.nh) continue;
      auto state = [&](int k) {
        return (k & 1 ? reinterpret_cast<const float*>(ring + (k >> 1) * kTiles * Y::kTile) : first + (k >> 1) * Y::kPart) +
               h * W;
      };
      // at most one state a warp; all their loads run at once
      float M = -INFINITY, L = 0.0f;
      float2 ml[NW];
      float4 y[NW];
      uint32_t x = set;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        ml[k] = make_float2(-INFINITY, 0.0f);
        y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (x) {
          const float* p = state(__ffs(x) - 1);
          ml[k] = *reinterpret_cast<const float2*>(p + HD);
          y[k] = *reinterpret_cast<const float4*>(p + d);
          M = fmaxf(M, ml[k].x);
        }
        x &= x - 1;
      }
      const float z = M == -INFINITY ? 0.0f : M;
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float e = exp2f(ml[k].x - z);
        add4(a, e, y[k]);
        L += e * ml[k].y;
      }
      if (w.seg0 >= 0 && w.seg0 + w.nblk <= n) {
        write_out(out + w.b * out_ld + static_cast<long long>(w.h0 + h) * HD,
                  lse ? lse + static_cast<long long>(w.b) * H + w.h0 + h : nullptr, M, L, a, d, vec);
      } else {
        float* part = parts_ws + static_cast<long long>(2 * cta + (w.seg0 >= 0 ? 1 : 0)) * Y::kPart + h * W;
        *reinterpret_cast<float4*>(part + d) = a;
        if (d == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(M, L);
      }
    }

    // ---- parts that cross CTAs, the run's first and last at most: the last CTA to finish joins the partial states
    const int e0 = __ffs(there) - 1, e1 = 31 - __clz(there);
    const Owner ends[2] = {sh.own[e0], sh.own[e1]};
    const bool one = ends[0].b == ends[1].b && ends[0].h0 == ends[1].h0;
    bool cross[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) cross[x] = (ends[x].seg0 < 0 || ends[x].seg0 + ends[x].nblk > n) && !(x && one);
    if (cross[0] || cross[1]) {
      __syncthreads();  // the ticket's release covers the whole CTA's states
      if (threadIdx.x < 2) {
        const Owner w = ends[threadIdx.x];
        bool last = false;
        if (cross[threadIdx.x]) {
          // the CTAs before this one and after it that have units of the part
          const int c0 = cta - (w.seg0 < 0 ? (per - 1 - w.seg0) / per : 0), c1 = cta + (w.seg0 + w.nblk - 1) / per;
          sh.c0[threadIdx.x] = c0;
          sh.np[threadIdx.x] = c1 - c0 + 1;
          last = ticket(&cnt[c0]) == c1 - c0;
          if (last) cnt[c0] = 0;
        }
        sh.last[threadIdx.x] = last;
      }
      __syncthreads();
      // A thread has four dimensions of a head and every other state, so that up to 16 states are loaded at once.
      for (int x = 0; x < 2; ++x) {
        if (!sh.last[x]) continue;
        const Owner w = ends[x];
        const int c0 = sh.c0[x], np = sh.np[x], half = lane >> 4;
        for (int i = warp * 16 + (lane & 15); i < w.nh * (HD / 4); i += Y::kThreads / 2) {  // whole warps go round
          constexpr int kDeep = 8;
          const int h = i / (HD / 4), d = i % (HD / 4) * 4;
          float M = -INFINITY, L = 0.0f;
          float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int k0 = 0; k0 < np; k0 += 2 * kDeep) {
            float4 y[kDeep];
            float2 ml[kDeep];
            float m = M;
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
              const int part = min(k0 + 2 * k + half, np - 1);  // the part-th CTA's state
              const float* p = parts_ws + static_cast<long long>(2 * (c0 + part) + (part == 0)) * Y::kPart + h * W;
              ml[k] = __ldcg(reinterpret_cast<const float2*>(p + HD));
              y[k] = __ldcg(reinterpret_cast<const float4*>(p + d));
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k) m = k0 + 2 * k + half < np ? fmaxf(m, ml[k].x) : m;
            const float z = m == -INFINITY ? 0.0f : m, e = exp2f(M - z);
            a = make_float4(a.x * e, a.y * e, a.z * e, a.w * e);
            L *= e;
            M = m;
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
              if (k0 + 2 * k + half < np) {
                const float e = exp2f(ml[k].x - z);
                add4(a, e, y[k]);
                L += e * ml[k].y;
              }
            }
          }
          const float mo = __shfl_xor_sync(0xffffffffu, M, 16), m = fmaxf(M, mo);
          const float e = exp2f(M - (m == -INFINITY ? 0.0f : m));
          a = make_float4(a.x * e, a.y * e, a.z * e, a.w * e);
          L *= e;
          a.x += __shfl_xor_sync(0xffffffffu, a.x, 16);
          a.y += __shfl_xor_sync(0xffffffffu, a.y, 16);
          a.z += __shfl_xor_sync(0xffffffffu, a.z, 16);
          a.w += __shfl_xor_sync(0xffffffffu, a.w, 16);
          L += __shfl_xor_sync(0xffffffffu, L, 16);
          if (half == 0)
            write_out(out + w.b * out_ld + static_cast<long long>(w.h0 + h) * HD,
                      lse ? lse + static_cast<long long>(w.b) * H + w.h0 + h : nullptr, m, L, a, d, vec);
        }
      }
    }
  }

  // ---- rows of the batch that attend nothing
  for (int b = cta; b < B; b += grid) {
    int lo, hi;
    span(pos, b, room, window, &lo, &hi);
    if (hi > lo) continue;
    for (int i = threadIdx.x; i < H * HD; i += Y::kThreads) from_f32(0.0f, out + b * out_ld + i);
    if (lse)
      for (int h = threadIdx.x; h < H; h += Y::kThreads) lse[static_cast<long long>(b) * H + h] = -INFINITY;
  }
}

// ----------------------------------------------------------------------------------------- host
static int check_kv(const char* what, const aib_paged_kv* c, Kv* o) {
  if (!c || !c->k || !c->v || c->pages <= 0 || c->KV <= 0) return fail(AIB_EINVAL, "%s: bad cache", what);
  if (c->HD != 64 && c->HD != 128) return fail(AIB_ENOTSUP, "%s: HD must be 64 or 128 (HD=%d)", what, c->HD);
  if (c->page <= 0 || (c->page & (c->page - 1)))
    return fail(AIB_EINVAL, "%s: rows per page must be a power of two (%d)", what, c->page);
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) ||
      ((c->page_stride | c->head_stride | c->row_stride) & 7))
    return fail(AIB_EINVAL, "%s: cache rows must start on 16-byte boundaries", what);
  // from the smallest stride on, every one steps over all that lies within it
  long long n[3] = {c->pages, c->KV, c->page}, st[3] = {c->page_stride, c->head_stride, c->row_stride};
  if (st[0] < st[1]) std::swap(st[0], st[1]), std::swap(n[0], n[1]);
  if (st[1] < st[2]) std::swap(st[1], st[2]), std::swap(n[1], n[2]);
  if (st[0] < st[1]) std::swap(st[0], st[1]), std::swap(n[0], n[1]);
  __int128 within = c->HD;
  bool apart = true;
  for (int i = 2; i >= 0; --i) {
    if (n[i] == 1) continue;
    apart = apart && st[i] >= within;
    within += static_cast<__int128>(n[i] - 1) * st[i];
  }
  if (!apart)
    return fail(AIB_EINVAL, "%s: cache rows overlap", what);
  *o = Kv{c->k, c->v, c->page_stride, c->head_stride, c->row_stride, c->pages, c->KV, __builtin_ctz(c->page)};
  return AIB_OK;
}

template <typename E>
static bool vec_rows(const Rows<E>& r) {  // whether four elements may be read at once
  return !r.p || (!(reinterpret_cast<uintptr_t>(r.p) % (4 * sizeof(E))) && !((r.ts | r.hs) & 3));
}

template <typename E>
static int append(const Kv& c, int HD, const int32_t* table, long long table_ld, int max_pages, const int64_t* pos,
                  const int32_t* cu, int B, int T, int H, Rows<const E> q, Rows<const E> k, Rows<const E> v, Rows<E> qo,
                  const uint16_t* qn, const uint16_t* kn, const float* inv, float eps, cudaStream_t s) {
  const int nv = H + 2 * c.KV;
  // A token's vectors go to as few warps as fill the GPU four times over (eight CTAs of eight warps an SM): a warp pays
  // for its token's angles once, but one warp alone is as slow as its loads one after the other.
  const int batch = kAppSteps * 256 / HD;
  const long long want = 4LL * 64 * sm_count();
  int parts = static_cast<int>(std::min<long long>((want + T - 1) / T, (nv + batch - 1) / batch));
  const int per = ((nv + parts - 1) / parts + batch - 1) / batch * batch;
  parts = (nv + per - 1) / per;
  const long long warps = static_cast<long long>(T) * parts;
  const dim3 grid(static_cast<unsigned>((warps + kAppWarps - 1) / kAppWarps));
  auto go = [&](auto kernel) {
    return launch(kernel, grid, dim3(32 * kAppWarps), 0, s, "aib_paged_append", c, table, table_ld, max_pages, pos, cu,
                  B, T, H, q, k, v, qo, qn, kn, inv, eps, parts, per);
  };
  if (vec_rows(q) && vec_rows(k) && vec_rows(v) && vec_rows(qo))
    return HD == 128 ? go(append_kernel<128, E, true>) : go(append_kernel<64, E, true>);
  return HD == 128 ? go(append_kernel<128, E, false>) : go(append_kernel<64, E, false>);
}

static int max_grid() { return std::min(kMaxGrid, sm_count()); }

static size_t attn_ws_bytes(int HD) {
  return kMaxGrid * sizeof(int) +
         static_cast<size_t>(2) * max_grid() * (HD == 128 ? Lay<128>::kPart : Lay<64>::kPart) * sizeof(float);
}

template <int HD>
static constexpr size_t smem_bytes() {
  return 1024 + Lay<HD>::kRing + Lay<HD>::kWarps * Lay<HD>::kPart * sizeof(float) + sizeof(Shared<HD>);
}

// Tensor map of the pool: boxes of HD elements (in halves of 128 bytes, swizzled) x the rows of a page, 32 at most.
static int pool_map(CUtensorMap* map, const uint16_t* p, const aib_paged_kv* c) {
  const uint64_t HD = c->HD, halves = HD / 64, page = c->page, KV = c->KV, pages = c->pages;
  // the stride of a dimension of one element means nothing, but it has to be a valid one
  const uint64_t sr = 2 * (page > 1 ? c->row_stride : HD), sh = 2 * (KV > 1 ? c->head_stride : HD),
                 sp = 2 * (pages > 1 ? c->page_stride : HD);
  const uint32_t rows = static_cast<uint32_t>(std::min(c->page, kBlk));
  if (halves == 1) {
    const uint64_t dims[4] = {64, page, KV, pages}, strides[3] = {sr, sh, sp};
    const uint32_t box[4] = {64, rows, 1, 1};
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 4, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const uint64_t dims[5] = {64, page, halves, KV, pages}, strides[4] = {sr, 128, sh, sp};
  const uint32_t box[5] = {64, rows, 2, 1, 1};
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 5, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int HD, typename E>
static int attend(const aib_paged_kv* c, const int32_t* table, long long table_ld, int room, const int64_t* pos, int B, int H,
                  const void* q, long long q_ld, void* out, long long out_ld, float* lse, long long window, float scale,
                  void* ws, cudaStream_t s) {
  const int G = H / c->KV, tiles = (G + GT - 1) / GT;
  // the shared-memory limit is raised once on each device (the query behind it costs more than the rest of a call)
  static std::atomic<uint64_t> raised{0};
  int dev = 0, rc = AIB_OK;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(raised.load(std::memory_order_relaxed) >> dev & 1)) {
    rc = allow_smem(attn_kernel<HD, E>, smem_bytes<HD>());
    if (!rc && dev < 64) raised.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  CUtensorMap kmap, vmap;
  if (!rc) rc = pool_map(&kmap, c->k, c);
  if (!rc) rc = pool_map(&vmap, c->v, c);
  if (rc) return rc;
  // no more CTAs than the longest sequences the table allows could fill
  const long long rows = window > 0 ? std::min<long long>(std::min<long long>(window, room) + kBlk - 1, room) : room;
  const long long units = static_cast<long long>(B) * c->KV * tiles * ((rows + kBlk - 1) / kBlk);
  const int grid = static_cast<int>(std::min<long long>(max_grid(), (units + Lay<HD>::kMinRun - 1) / Lay<HD>::kMinRun));
  return launch(attn_kernel<HD, E>, dim3(grid), dim3(Lay<HD>::kThreads), smem_bytes<HD>(), s, "aib_paged_attn", kmap, vmap,
                c->pages, c->KV, __builtin_ctz(c->page), table, table_ld, room, pos, B, H, static_cast<const E*>(q),
                q_ld, static_cast<E*>(out), out_ld, lse, window, scale, static_cast<int*>(ws),
                reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kMaxGrid * sizeof(int)));
}

}  // namespace paged
}  // namespace aib

using namespace aib;

extern "C" {

int aib_paged_append(const aib_paged_kv* cache, const int32_t* table, int64_t table_ld, int max_pages,
                     const int64_t* pos, const int32_t* cu, int B, int T, int H, const void* q, int64_t q_ts,
                     int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                     void* q_out, int64_t qo_ts, int64_t qo_hs, int dtype, const uint16_t* qn, const uint16_t* kn,
                     const float* inv, float eps, void* stream) {
  paged::Kv c;
  const int rc = paged::check_kv("aib_paged_append", cache, &c);
  if (rc) return rc;
  if (!table || !pos || !k || !v || B <= 0 || T <= 0 || max_pages <= 0 || table_ld < 0 || (dtype != 0 && dtype != 1))
    return fail(AIB_EINVAL, "aib_paged_append: bad arguments");
  if (!cu && T != B) return fail(AIB_EINVAL, "aib_paged_append: without cu, T must be B (T=%d B=%d)", T, B);
  if (H < 0 || (H > 0) != (q != nullptr) || (H > 0) != (q_out != nullptr))
    return fail(AIB_EINVAL, "aib_paged_append: q and q_out go with H > 0");
  const size_t es = dtype == 0 ? 4 : 2;
  if (!aligned(es, q, k, v, q_out) || !aligned(4, table, cu, inv) || !aligned(8, pos) || !aligned(2, qn, kn))
    return fail(AIB_EINVAL, "aib_paged_append: every argument must be aligned to its elements");
  if (static_cast<long long>(T) * (H + 2LL * c.KV) > 0x7fffffffLL)
    return fail(AIB_ENOTSUP, "aib_paged_append: T * (H + 2 KV) must fit 31 bits");
  if (H > 0) {
    auto rows = [&](const void* p, int heads, int64_t ts, int64_t hs) {
      return Rows2{reinterpret_cast<uintptr_t>(p), static_cast<long long>(cache->HD * es), {T, heads}, {ts, hs}, es};
    };
    const Rows2 to = rows(q_out, H, qo_ts, qo_hs);
    const bool same = q_out == q && (T == 1 || qo_ts == q_ts) && (H == 1 || qo_hs == q_hs);
    if (!rows_apart(to) || (!same && rows_meet(to, rows(q, H, q_ts, q_hs))) || rows_meet(to, rows(k, c.KV, k_ts, k_hs)) ||
        rows_meet(to, rows(v, c.KV, v_ts, v_hs)))
      return fail(AIB_EINVAL, "aib_paged_append: the rows of q_out must lie apart, and be q's or share no memory with q, k and v");
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto e) {
    using E = decltype(e);
    return paged::append<E>(c, cache->HD, table, table_ld, max_pages, pos, cu, B, T, H,
                            paged::Rows<const E>{static_cast<const E*>(q), q_ts, q_hs},
                            paged::Rows<const E>{static_cast<const E*>(k), k_ts, k_hs},
                            paged::Rows<const E>{static_cast<const E*>(v), v_ts, v_hs},
                            paged::Rows<E>{static_cast<E*>(q_out), qo_ts, qo_hs}, qn, kn, inv, eps, s);
  };
  return dtype == 0 ? go(float()) : go(uint16_t());
}

size_t aib_paged_attn_workspace(int B, int H, int KV, int HD) {
  if (B <= 0 || H <= 0 || KV <= 0 || H % KV || (HD != 64 && HD != 128)) return 0;
  return paged::attn_ws_bytes(HD);
}

int aib_paged_attn(const aib_paged_kv* cache, const int32_t* table, int64_t table_ld, int max_pages,
                   const int64_t* pos, int B, int H, const void* q, int64_t q_ld, void* out, int64_t out_ld, int dtype, float* lse,
                   int64_t window, float scale, void* ws, size_t ws_bytes, void* stream) {
  paged::Kv c;
  const int rc = paged::check_kv("aib_paged_attn", cache, &c);
  if (rc) return rc;
  if (!table || !pos || !q || !out || B <= 0 || max_pages <= 0 || table_ld < 0 || window < 0 ||
      (dtype != 0 && dtype != 1) || H <= 0 || H % c.KV || q_ld < 0 || out_ld < 0)
    return fail(AIB_EINVAL, "aib_paged_attn: bad arguments");
  const size_t es = dtype == 0 ? 4 : 2;
  if (!aligned(es, q, out) || !aligned(4, table, lse) || !aligned(8, pos))
    return fail(AIB_EINVAL, "aib_paged_attn: every argument must be aligned to its elements");
  if (B > paged::kMaxBatch) return fail(AIB_ENOTSUP, "aib_paged_attn: at most %d sequences (%d)", paged::kMaxBatch, B);
  const long long room = static_cast<long long>(max_pages) * cache->page;
  const long long tiles = (H / c.KV + paged::GT - 1) / paged::GT, units = (room + paged::kBlk - 1) / paged::kBlk;
  if (room > 0x7fffff00LL || static_cast<long long>(H) * cache->HD > 0x7fffffffLL ||
      units * tiles > (0x7fffffffLL << 6) / B / c.KV)
    return fail(AIB_ENOTSUP, "aib_paged_attn: max_pages * page and H * HD must fit 31 bits, all the rows of the batch 42");
  const size_t need = paged::attn_ws_bytes(cache->HD);
  if (!ws || ws_bytes < need)
    return fail(AIB_EWORKSPACE, "aib_paged_attn: workspace %zu < %zu bytes", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) & 15) return fail(AIB_EINVAL, "aib_paged_attn: the workspace must be 16-byte aligned");
  const long long row = static_cast<long long>(H) * cache->HD * es;
  const Rows2 from{reinterpret_cast<uintptr_t>(q), row, {B, 1}, {q_ld, 0}, es},
      to{reinterpret_cast<uintptr_t>(out), row, {B, 1}, {out_ld, 0}, es},
      sums{reinterpret_cast<uintptr_t>(lse), 4LL * B * H, {lse ? 1 : 0, 1}, {0, 0}, 1};
  if (!rows_apart(to) || rows_meet(to, from) || rows_meet(sums, from) || rows_meet(sums, to))
    return fail(AIB_EINVAL, "aib_paged_attn: the rows of out must lie apart, and out, lse and q share no memory");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto fn) {
    return fn(cache, table, table_ld, static_cast<int>(room), pos, B, H, q, q_ld, out, out_ld, lse, window, scale, ws, s);
  };
  if (cache->HD == 128) return dtype == 0 ? go(paged::attend<128, float>) : go(paged::attend<128, uint16_t>);
  return dtype == 0 ? go(paged::attend<64, float>) : go(paged::attend<64, uint16_t>);
}

}  // extern "C"
