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
// out = sum_j softmax_j(scale q.k_j) v_j in one pass over the rows with a running maximum and sum (in base 2).
//
// Split: the work is a line of units, a unit being 32 cached rows (from a multiple of 32) of one (sequence, key head,
// tile of 8 query heads), and every CTA, one an SM, takes an equal run of it, so the load does not depend on how ragged
// the lengths are and the host need not know them (a captured step keeps its grid while the sequences grow). Where a
// (sequence, head) crosses CTAs each writes a partial state, and the last one to finish (a ticket; nobody waits) joins
// them in order, so that the sums do not depend on timing.
//
// Roles in a CTA: one warp looks up pages and starts the tensor copies of K and V pages into a ring of stages; eight
// warps take the units in turn, each with its own running state; three warps join the eight states
// of a finished (sequence, head) and write it, while the others are already at the next one. The copies land in the
// 128-byte swizzle, so the eight row addresses of an ldmatrix hit different banks.
//
// Masked rows (outside the span, or on a page outside the pool) get weight 0 and their V rows are cleared in shared
// memory, whatever the cache holds there; boxes without a row to attend are not fetched.
//
// The few query rows (at most 8 a tile) go through mma.sync as the 8 columns: the kernel is bound by the cache's bytes,
// and the tensor cores are far from their limit (3 products of 16 x 8 x 16 a 16 x 16 piece of K or V). fp32 rows enter as
// three bf16 parts and so do their weights (24 bits, as good as fp32 products); bf16 rows are exact as they are, and
// their weights take two parts (16 bits, 2^-8 of the output's own rounding). An mma chops its sums where an fp32 addition
// rounds, so no long chain runs through one accumulator: the rows' running sums are added outside.
constexpr int GT = 8;       // query heads of a group served together (the columns of an mma)
constexpr int kCons = 8;    // warps that take units
constexpr int kEpi = 3;     // warps that join states
constexpr int kThreads = 32 * (1 + kEpi + kCons);
constexpr int kBlk = 32;    // rows of a unit
constexpr int kMinRun = 4;  // units of a CTA's run at least
constexpr int kMaxBatch = 4096;
constexpr int kMaxGrid = 1024;

template <int HD>
struct Lay {
  static constexpr int kTile = kBlk * HD * 2;           // the K or V rows of a unit: its boxes one after the other
  static constexpr int kStages = HD == 128 ? 10 : 22;
  static_assert(kStages >= kCons, "");
  static constexpr int kW = HD + 2;                     // a head's sums, its maximum, its sum of weights
  static constexpr int kPart = GT * kW;                 // floats of a state
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kBytes = 1024 + kRing + kCons * kPart * 4 + kCons * GT * kBlk * 4;
};

template <int N>
AIB_DEV void split_pair(float lo, float hi, uint32_t* w) {  // lo, hi as N bf16 parts each, (hi << 16) | lo
#pragma unroll
  for (int k = 0; k < N; ++k) {
    w[k] = bf16x2_rn(lo, hi);
    lo -= __uint_as_float(w[k] << 16);
    hi -= __uint_as_float(w[k] & 0xFFFF0000u);
  }
}
// Rows [row, row + box) of head kvh in page id: [HD / 64][box][64] elements in shared memory, 128-byte swizzle.
template <int HD>
AIB_DEV void tma_load(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int row, int kvh, int id) {
  if (HD == 128)
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(kvh), "r"(id)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(kvh), "r"(id)
        : "memory");
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

// A place in a CTA's run: sequence b, its part s (key head * tiles + tile), whose units are [seg0, seg0 + nblk), counted
// from the run's first unit (seg0 is negative where the part began in an earlier run).
struct Cursor {
  int seg0, nblk, b, s, lo, hi;
};
struct Line {
  const int64_t* pos;
  long long window;
  int B, room, parts;
};
AIB_DEV void enter(Cursor& c, const Line& l) {
  span(l.pos, c.b, l.room, l.window, &c.lo, &c.hi);
  c.nblk = units_of(c.lo, c.hi);
}
AIB_DEV void seek(Cursor& c, const Line& l, int u) {  // forward to the part that holds unit u
  while (u - c.seg0 >= c.nblk) {
    c.seg0 += c.nblk;
    if (++c.s == l.parts) {
      c.s = 0;
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

// Two neighbouring outputs (dimensions d, d + 1) of a head from its sums.
template <typename E>
AIB_DEV void write_out(E* out, float* lse, float M, float L, float2 a, int d) {
  float o[2] = {M == -INFINITY ? 0.0f : a.x / L, M == -INFINITY ? 0.0f : a.y / L};
  store_per<1>(out + d, 0, o);
  store_per<1>(out + d + 1, 0, o + 1);
  if (lse && d == 0) *lse = M == -INFINITY ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

template <int HD>
struct AttnShared {
  uint64_t full_k[Lay<HD>::kStages], full_v[Lay<HD>::kStages], empty[Lay<HD>::kStages];
  uint64_t st_full[kCons], st_free[kCons];
  uint32_t mask[Lay<HD>::kStages];  // rows of the unit that are attended
  long long wtot[kThreads / 32], base;
  int b, last, fail[kEpi];
  float M[GT], L[GT];
};

template <int HD, typename E>
__global__ void __launch_bounds__(kThreads, 1)
    attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, int pages, int KV,
                int page_shift, const int32_t* __restrict__ table, int table_ld, int room,
                const int64_t* __restrict__ pos, int B, int H, const E* __restrict__ q, long long q_ld,
                E* __restrict__ out, long long out_ld, float* __restrict__ lse, long long window, float scale, int* cnt,
                float* parts_ws) {
  using L_ = Lay<HD>;
  constexpr int PQ = sizeof(E) == 4 ? 3 : 1, PP = sizeof(E) == 4 ? 3 : 2;
  constexpr int NT = HD / 16, W = L_::kW, NS = L_::kStages;
  extern __shared__ uint8_t dyn[];
  __shared__ AttnShared<HD> sh;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~static_cast<uintptr_t>(1023));
  float* state = reinterpret_cast<float*>(ring + L_::kRing);
  float* pws = state + kCons * L_::kPart;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cta = blockIdx.x, grid = gridDim.x;
  const int G = H / KV, tiles = (G + GT - 1) / GT;
  const Line line{pos, window, B, room, KV * tiles};
  if (threadIdx.x < NS) {
    mbar_init(&sh.full_k[threadIdx.x], 1);
    mbar_init(&sh.full_v[threadIdx.x], 1);
    mbar_init(&sh.empty[threadIdx.x], 1);
  }
  if (threadIdx.x < kCons) {
    mbar_init(&sh.st_full[threadIdx.x], 1);
    mbar_init(&sh.st_free[threadIdx.x], kEpi);
  }
  if (warp == 0) fence_mbar_init();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  pdl_wait();
  pdl_trigger();

  // ---- this CTA's run, n units from u0: a sum over the sequences' units, every thread over a few of them
  const int cb = (B + kThreads - 1) / kThreads, b_lo = min(B, static_cast<int>(threadIdx.x) * cb),
            b_hi = min(B, b_lo + cb);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    int lo, hi;
    if (!span(pos, b, room, window, &lo, &hi) && cta == 0) set_status(AIB_DEV_BAD_POS);
    mine += units_of(lo, hi);
  }
  mine *= line.parts;
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
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.wtot[w];
    total += sh.wtot[w];
  }
  const long long per = max(static_cast<long long>(kMinRun), (total + grid - 1) / grid);
  const long long u0 = cta * per;
  const int n = static_cast<int>(max(0LL, min(total - u0, per)));  // units of the run
  if (n > 0) {
    long long base = before + incl - mine;
    if (u0 >= base && u0 < base + mine) {
      for (int b = b_lo; b < b_hi; ++b) {
        int lo, hi;
        span(pos, b, room, window, &lo, &hi);
        const long long n = static_cast<long long>(units_of(lo, hi)) * line.parts;
        if (u0 < base + n) {
          sh.b = b;
          sh.base = base;
          break;
        }
        base += n;
      }
    }
  }
  __syncthreads();
  Cursor C{0, 1, 0, 0, 0, 0};
  if (n > 0) {
    C.b = sh.b;
    enter(C, line);
    C.s = static_cast<int>((u0 - sh.base) / C.nblk);
    C.seg0 = -static_cast<int>((u0 - sh.base) % C.nblk);
  }

  if (warp <= kEpi) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0) {
      // -------------------------------------------------------------------- pages -> ring of stages
      // A lane stands for a box of rows of one page (at most 32 rows): it finds its unit, looks up its page and starts
      // its copies, so what finding costs is shared by all the units of a batch of 32 boxes, and the next batch's
      // look-ups run while this one's copies start.
      const int box = min(kBlk, 1 << page_shift), nbox = kBlk / box, batch = 32 / nbox;  // units of a batch
      const int bx = lane & (nbox - 1), bu = lane / nbox;                                // the lane's box, its unit
      struct Look {
        int id, row, kvh;
        uint32_t rows;  // the box's rows that are attended, as bits of the unit
      };
      auto look_up = [&](int i) {
        Look k{-1, 0, 0, 0};
        if (i + bu < n) {
          seek(C, line, i + bu);
          const int j0 = (C.lo & ~(kBlk - 1)) + (i + bu - C.seg0) * kBlk, a = j0 + bx * box;
          const int r0 = max(a, C.lo) - j0, r1 = min(a + box, C.hi) - j0;  // within the unit
          k.kvh = C.s / tiles;
          k.row = a & ((1 << page_shift) - 1);
          if (r0 < r1) {
            k.rows = (0xffffffffu >> (32 - (r1 - r0))) << r0;
            k.id = table[static_cast<long long>(C.b) * table_ld + (a >> page_shift)];
          }
        }
        return k;
      };
      const uint32_t ring32 = smem_u32(ring) + bx * box * HD * 2;
      Look next = look_up(0);
      int st = 0, ph = 1, i = 0;
      bool ok = true;
      while (i < n && ok) {
        Look k = next;
        if (k.rows && (k.id < 0 || k.id >= pages)) {
          set_status(AIB_DEV_BAD_PAGE);
          k.rows = 0;
        }
        uint32_t mask = k.rows, bytes = k.rows ? box * HD * 2 : 0;
        for (int o = 1; o < nbox; o <<= 1) {
          mask |= __shfl_xor_sync(0xffffffffu, mask, o);
          bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
        }
        next = look_up(i + batch);
        for (int u = 0; u < batch && i < n; ++u, ++i) {
          ok = mbar_wait(&sh.empty[st], ph, AIB_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          if (lane == u * nbox) {
            sh.mask[st] = mask;
            mbar_arrive_expect_tx(&sh.full_k[st], bytes);
            mbar_arrive_expect_tx(&sh.full_v[st], bytes);
          }
          __syncwarp();
          if (bu == u && k.rows) {
            const uint32_t dst = ring32 + st * 2 * L_::kTile;
            tma_load<HD>(dst, &kmap, &sh.full_k[st], k.row, k.kvh, k.id);
            tma_load<HD>(dst + L_::kTile, &vmap, &sh.full_v[st], k.row, k.kvh, k.id);
          }
          if (++st == NS) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      // The consumers wait for every copy before they end. After a wait that ran out they may not, so this warp does.
      if (!ok)
        for (int k = 0; k < NS && --i >= 0; ++k) {
          mbar_wait(&sh.full_k[i % NS], i / NS & 1, AIB_DEV_TIMEOUT_FULL);
          mbar_wait(&sh.full_v[i % NS], i / NS & 1, AIB_DEV_TIMEOUT_FULL);
        }
    } else {
      // ----------------------------------------------------------------- states -> outputs, partials
      constexpr int kEt = 32 * kEpi;
      const int et = threadIdx.x - 32, ew = warp - 1;
      uint32_t phase = 0;
      while (n > 0) {
        const int beg = max(0, C.seg0), end = min(n, C.seg0 + C.nblk);
        const int h0 = (C.s / tiles) * G + (C.s % tiles) * GT, nh = min(GT, G - (C.s % tiles) * GT);
        const int nw = min(kCons, end - beg), w0 = beg % kCons;
        bool ok = true;
        for (int k = 0; k < nw; ++k) {
          const int w = (w0 + k) % kCons;
          ok = ok && mbar_wait(&sh.st_full[w], phase >> w & 1, AIB_DEV_TIMEOUT_FULL);
          phase ^= 1u << w;
        }
        if (lane == 0) sh.fail[ew] = !ok;
        named_sync(1, kEt);
        bool failed = false;
#pragma unroll
        for (int k = 0; k < kEpi; ++k) failed = failed || sh.fail[k];
        if (failed) break;
        const bool whole = C.seg0 >= 0 && C.seg0 + C.nblk <= n;
        float* part = parts_ws + static_cast<long long>(2 * cta + (C.seg0 >= 0 ? 1 : 0)) * L_::kPart;
        E* orow = out + C.b * out_ld + static_cast<long long>(h0) * HD;
        float* lrow = lse ? lse + static_cast<long long>(C.b) * H + h0 : nullptr;
        for (int i = et; i < nh * (HD / 2); i += kEt) {
          const int h = i / (HD / 2), d = i % (HD / 2) * 2;
          float M = -INFINITY, L = 0.0f;
          float2 a = make_float2(0.0f, 0.0f);
          for (int k = 0; k < nw; ++k) M = fmaxf(M, state[(w0 + k) % kCons * L_::kPart + h * W + HD]);
          const float z = M == -INFINITY ? 0.0f : M;
          for (int k = 0; k < nw; ++k) {
            const float* x = state + (w0 + k) % kCons * L_::kPart + h * W;
            const float e = exp2f(x[HD] - z);
            const float2 y = *reinterpret_cast<const float2*>(x + d);
            L += e * x[HD + 1];
            a.x += e * y.x;
            a.y += e * y.y;
          }
          if (whole) {
            write_out(orow + h * HD, lrow ? lrow + h : nullptr, M, L, a, d);
          } else {
            *reinterpret_cast<float2*>(part + h * W + d) = a;
            if (d == 0) *reinterpret_cast<float2*>(part + h * W + HD) = make_float2(M, L);
          }
        }
        __syncwarp();
        if (lane == 0)
          for (int k = 0; k < nw; ++k) mbar_arrive(&sh.st_free[(w0 + k) % kCons]);
        if (!whole) {
          // the CTAs that share this part: the last one joins their states, in order
          const int c0 = static_cast<int>((u0 + C.seg0) / per), c1 = static_cast<int>((u0 + C.seg0 + C.nblk - 1) / per);
          __threadfence();
          named_sync(1, kEt);
          if (et == 0) sh.last = atomicAdd(&cnt[c0], 1) == c1 - c0;
          named_sync(1, kEt);
          if (sh.last) {
            __threadfence();
            auto part_of = [&](int k) {  // the k-th CTA's state
              return parts_ws + static_cast<long long>(2 * (c0 + k) + (k == 0)) * L_::kPart;
            };
            const int np = c1 - c0 + 1;
            for (int h = ew; h < nh; h += kEpi) {
              float M = -INFINITY, L = 0.0f;
              for (int k = lane; k < np; k += 32) M = fmaxf(M, __ldcg(part_of(k) + h * W + HD));
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
              const float z = M == -INFINITY ? 0.0f : M;
              for (int k = lane; k < np; k += 32) {
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_of(k) + h * W + HD));
                L += exp2f(ml.x - z) * ml.y;
              }
              L = warp_sum(L);
              if (lane == 0) {
                sh.M[h] = M;
                sh.L[h] = L;
              }
            }
            named_sync(1, kEt);
            for (int i = et; i < nh * (HD / 2); i += kEt) {
              const int h = i / (HD / 2), d = i % (HD / 2) * 2;
              const float M = sh.M[h], z = M == -INFINITY ? 0.0f : M;
              float2 a = make_float2(0.0f, 0.0f);
#pragma unroll 8
              for (int k = 0; k < np; ++k) {
                const float* x = part_of(k) + h * W;
                const float e = exp2f(__ldcg(x + HD) - z);
                const float2 y = __ldcg(reinterpret_cast<const float2*>(x + d));
                a.x += e * y.x;
                a.y += e * y.y;
              }
              write_out(orow + h * HD, lrow ? lrow + h : nullptr, M, sh.L[h], a, d);
            }
            if (et == 0) cnt[c0] = 0;
          }
        }
        if (end >= n) break;
        seek(C, line, end);
      }
      // rows of the batch that attend nothing
      for (int b = cta; b < B; b += grid) {
        int lo, hi;
        span(pos, b, room, window, &lo, &hi);
        if (hi > lo) continue;
        const float zero = 0.0f;
        for (int i = et; i < H * HD; i += kEt) store_per<1>(out + b * out_ld + i, 0, &zero);
        if (lse)
          for (int h = et; h < H; h += kEt) lse[static_cast<long long>(b) * H + h] = -INFINITY;
      }
    }
    return;
  }

  // ------------------------------------------------------------------------------------ units -> states
  asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
  const int cw = warp - 1 - kEpi, g = lane >> 2, t = lane & 3;
  const float sl = scale * 1.4426950408889634f;
  float* pw = pws + cw * GT * kBlk;
  float* mine_st = state + cw * L_::kPart;
  const uint32_t ring32 = smem_u32(ring);
  // ldmatrix rows: box by box, [HD / 64][box][128 bytes]. The 16-byte chunk c of the 128 bytes at address a lies in chunk
  // c ^ (a / 128 % 8): `place` gives a with that number in the chunk's bits, to be combined with c by one xor.
  const int box_shift = min(5, page_shift);
  auto place = [&](int row, int half) {
    const uint32_t a = ((row >> box_shift << box_shift) * (HD / 64) + (half << box_shift) + (row & ((1 << box_shift) - 1))) * 128;
    return a | ((a >> 7 & 7) << 4);
  };
  const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kcol = lane >> 4;       // A tile of K rows: row, chunk
  const int vr = (lane & 7) + (lane >> 4) * 8, vcol = (lane >> 3) & 1;       // V tile, transposed load
  uint32_t ka[2][HD / 64], va[2][HD / 64];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) {
      ka[m][h] = place(m * 16 + kr, h) ^ kcol << 4;
      va[m][h] = place(m * 16 + vr, h) ^ vcol << 4;
    }
  uint32_t free_phase = 1;
  int st = cw % NS, ph = 0;
  while (n > 0) {
    const int beg = max(0, C.seg0), end = min(n, C.seg0 + C.nblk);
    const int h0 = (C.s / tiles) * G + (C.s % tiles) * GT, nh = min(GT, G - (C.s % tiles) * GT);
    int u = beg + ((cw - beg) & (kCons - 1));
    if (u < end) {
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
      float acc[NT][4];
#pragma unroll
      for (int d = 0; d < NT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.0f;
      uint32_t bq[NT][PQ][2];  // q of head g, dimensions 16 s + 2t, +1 and +8, +9
      const E* qr = q + C.b * q_ld + static_cast<long long>(h0 + min(g, nh - 1)) * HD + 2 * t;
#pragma unroll
      for (int s = 0; s < NT; ++s) {
        float x[4];
        load_per<1>(qr + 16 * s, 0, x);
        load_per<1>(qr + 16 * s + 1, 0, x + 1);
        load_per<1>(qr + 16 * s + 8, 0, x + 2);
        load_per<1>(qr + 16 * s + 9, 0, x + 3);
        uint32_t w0[PQ], w1[PQ];
        split_pair<PQ>(x[0], x[1], w0);
        split_pair<PQ>(x[2], x[3], w1);
#pragma unroll
        for (int k = 0; k < PQ; ++k) bq[s][k][0] = w0[k], bq[s][k][1] = w1[k];
      }
      for (; u < end; u += kCons) {
        const uint32_t kt = ring32 + st * 2 * L_::kTile, vt = kt + L_::kTile;
        // A parity tells a phase from its neighbours only: this warp may be a whole round ahead of the one that has the
        // stage's previous unit, so it waits for that one's release first. (The release before it is certain: the copying
        // warp took it before it started this warp's last unit.)
        if (!mbar_wait(&sh.empty[st], ph ^ 1, AIB_DEV_TIMEOUT_EMPTY)) return;
        if (!mbar_wait(&sh.full_k[st], ph, AIB_DEV_TIMEOUT_FULL)) return;
        const uint32_t vm = sh.mask[st];
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
        // weights: sc[mt][0/1] are heads 2t, 2t+1 at row mt*16 + g, sc[mt][2/3] at row mt*16 + g + 8
        float s0[4], s1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = vm >> ((i >> 1) * 16 + g + (i & 1) * 8) & 1;
          s0[i] = ok ? sc[i >> 1][(i & 1) * 2] * sl : -INFINITY;
          s1[i] = ok ? sc[i >> 1][(i & 1) * 2 + 1] * sl : -INFINITY;
        }
        float b0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3])), b1 = fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, o));
          b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, o));
        }
        const float n0 = fmaxf(m0, b0), n1 = fmaxf(m1, b1);
        const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;  // no row so far: weights 0
        float q0 = 0.0f, q1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (i >> 1) * 16 + g + (i & 1) * 8;
          const float p0 = exp2f(s0[i] - z0), p1 = exp2f(s1[i] - z1);
          q0 += p0;
          q1 += p1;
          pw[2 * t * kBlk + row] = p0;
          pw[(2 * t + 1) * kBlk + row] = p1;
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          q0 += __shfl_xor_sync(0xffffffffu, q0, o);
          q1 += __shfl_xor_sync(0xffffffffu, q1, o);
        }
        const float al0 = exp2f(m0 - z0), al1 = exp2f(m1 - z1);
        l0 = l0 * al0 + q0;
        l1 = l1 * al1 + q1;
        m0 = n0;
        m1 = n1;
        __syncwarp();
        uint32_t bp[2][PP][2];  // weights of head g at rows 16 s + 2t, +1 and +8, +9
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float2 lo = *reinterpret_cast<const float2*>(pw + g * kBlk + s * 16 + 2 * t);
          const float2 hi = *reinterpret_cast<const float2*>(pw + g * kBlk + s * 16 + 2 * t + 8);
          uint32_t w0[PP], w1[PP];
          split_pair<PP>(lo.x, lo.y, w0);
          split_pair<PP>(hi.x, hi.y, w1);
#pragma unroll
          for (int k = 0; k < PP; ++k) bp[s][k][0] = w0[k], bp[s][k][1] = w1[k];
        }
        if (!mbar_wait(&sh.full_v[st], ph, AIB_DEV_TIMEOUT_FULL)) return;
        if (vm != 0xffffffffu) {  // clear the V rows that are not attended (the copies' next write comes after this)
          if (!(vm >> lane & 1)) {
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
              uint4* row = reinterpret_cast<uint4*>(ring + st * 2 * L_::kTile + L_::kTile + (place(lane, h) & ~127u));
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
            for (int k = PP - 1; k >= 0; --k) mma_bf16(x, a0, a1, a2, a3, bp[s][k][0], bp[s][k][1]);
          }
          acc[d][0] = acc[d][0] * al0 + x[0];
          acc[d][1] = acc[d][1] * al1 + x[1];
          acc[d][2] = acc[d][2] * al0 + x[2];
          acc[d][3] = acc[d][3] * al1 + x[3];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[st]);
        st += kCons;
        if (st >= NS) {
          st -= NS;
          ph ^= 1;
        }
      }
      if (!mbar_wait(&sh.st_free[cw], free_phase, AIB_DEV_TIMEOUT_EMPTY)) return;
      free_phase ^= 1;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float* dst = mine_st + (2 * t + hh) * W;
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
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.st_full[cw]);
    }
    if (end >= n) break;
    seek(C, line, end);
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

static int max_grid() { return std::min(kMaxGrid, sm_count()); }

static size_t attn_ws_bytes(int HD) {
  return kMaxGrid * sizeof(int) +
         static_cast<size_t>(2) * max_grid() * (HD == 128 ? Lay<128>::kPart : Lay<64>::kPart) * sizeof(float);
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
static int attend(const aib_paged_kv* c, const int32_t* table, int table_ld, int room, const int64_t* pos, int B, int H,
                  const void* q, long long q_ld, void* out, long long out_ld, float* lse, long long window, float scale,
                  void* ws, cudaStream_t s) {
  const int G = H / c->KV, tiles = (G + GT - 1) / GT;
  int rc = allow_smem(attn_kernel<HD, E>, Lay<HD>::kBytes);
  CUtensorMap kmap, vmap;
  if (!rc) rc = pool_map(&kmap, c->k, c);
  if (!rc) rc = pool_map(&vmap, c->v, c);
  if (rc) return rc;
  // no more CTAs than the longest sequences the table allows could fill
  const long long rows = window > 0 ? std::min<long long>(window + kBlk - 1, room) : room;
  const long long units = static_cast<long long>(B) * c->KV * tiles * ((rows + kBlk - 1) / kBlk);
  const int grid = static_cast<int>(std::min<long long>(max_grid(), (units + kMinRun - 1) / kMinRun));
  return launch(attn_kernel<HD, E>, dim3(grid), dim3(kThreads), Lay<HD>::kBytes, s, "aib_paged_attn", kmap, vmap,
                c->pages, c->KV, __builtin_ctz(c->page), table, table_ld, room, pos, B, H, static_cast<const E*>(q),
                q_ld, static_cast<E*>(out), out_ld, lse, window, scale, static_cast<int*>(ws),
                reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kMaxGrid * sizeof(int)));
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
  return paged::attn_ws_bytes(HD);
}

int aib_paged_attn(const aib_paged_kv* cache, const int32_t* table, int table_ld, int max_pages, const int64_t* pos,
                   int B, int H, const void* q, int64_t q_ld, void* out, int64_t out_ld, int dtype, float* lse,
                   int64_t window, float scale, void* ws, size_t ws_bytes, void* stream) {
  paged::Kv c;
  const int rc = paged::check_kv("aib_paged_attn", cache, &c);
  if (rc) return rc;
  if (!table || !pos || !q || !out || B <= 0 || max_pages <= 0 || table_ld < 0 || window < 0 ||
      (dtype != 0 && dtype != 1) || H <= 0 || H % c.KV || q_ld < 0 || out_ld < 0)
    return fail(AIB_EINVAL, "aib_paged_attn: bad arguments");
  if (B > paged::kMaxBatch) return fail(AIB_ENOTSUP, "aib_paged_attn: at most %d sequences (%d)", paged::kMaxBatch, B);
  const long long room = static_cast<long long>(max_pages) * cache->page;
  if (room > 0x7fffffffLL || static_cast<long long>(H) * cache->HD > 0x7fffffffLL)
    return fail(AIB_ENOTSUP, "aib_paged_attn: max_pages * page and H * HD must fit 31 bits");
  const size_t need = paged::attn_ws_bytes(cache->HD);
  if (!ws || ws_bytes < need)
    return fail(AIB_EWORKSPACE, "aib_paged_attn: workspace %zu < %zu bytes", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) & 15) return fail(AIB_EINVAL, "aib_paged_attn: the workspace must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto fn) {
    return fn(cache, table, table_ld, static_cast<int>(room), pos, B, H, q, q_ld, out, out_ld, lse, window, scale, ws, s);
  };
  if (cache->HD == 128) return dtype == 0 ? go(paged::attend<128, float>) : go(paged::attend<128, uint16_t>);
  return dtype == 0 ? go(paged::attend<64, float>) : go(paged::attend<64, uint16_t>);
}

}  // extern "C"
