// Library-wide host runtime: error messages, PDL switch, device status word, tensor-map encoding.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <set>
#include <utility>
#include "common.cuh"

namespace aib {
namespace attn {
extern int g_cluster_sizes;  // attn.cu
}
namespace gemv {
extern int g_variant;  // gemv.cu
}

static thread_local char t_err[512] = {0};
static int g_pdl = 1;

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(t_err, sizeof(t_err), fmt, ap);
  va_end(ap);
  return code;
}

bool pdl_enabled() { return g_pdl != 0; }

int sm_count(int device) {
  static int cache[64] = {0};
  if (device < 0 && cudaGetDevice(&device) != cudaSuccess) return 148;
  if (device >= 64) device = 63;
  if (!cache[device]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
    cache[device] = n;
  }
  return cache[device];
}

bool smem_raised(const void* kernel, int device, bool record) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> seen;
  std::lock_guard<std::mutex> lock(mu);
  if (record) seen.insert({kernel, device});
  return seen.count({kernel, device}) != 0;
}

namespace {
typedef __int128 wide;  // strides are the caller's numbers: no product of them may wrap
struct Grid2 {
  wide base, width, n[2], s[2];
  wide last() const { return base + width + (n[0] - 1) * s[0] + (n[1] - 1) * s[1]; }
};
// Strides positive and, where rows lie end to end, the rows joined; dimension 0 has the larger stride. `once`: rows
// that repeat (stride 0) count once.
Grid2 canonical(const Rows2& r, bool once) {
  const wide unit = r.unit;
  Grid2 g{static_cast<wide>(r.base), r.width, {r.n[0], r.n[1]}, {r.s[0] * unit, r.s[1] * unit}};
  for (int i = 0; i < 2; ++i) {
    if (g.s[i] < 0) {
      g.base += g.s[i] * (g.n[i] - 1);
      g.s[i] = -g.s[i];
    }
    if (g.n[i] == 1 || (once && g.s[i] == 0)) g.n[i] = 1, g.s[i] = 0;
  }
  if (g.s[0] < g.s[1]) std::swap(g.n[0], g.n[1]), std::swap(g.s[0], g.s[1]);
  for (int i = 1; i >= 0; --i)
    if (g.n[i] > 1 && g.s[i] == g.width) g.width *= g.n[i], g.n[i] = 1, g.s[i] = 0;
  if (g.s[0] < g.s[1]) std::swap(g.n[0], g.n[1]), std::swap(g.s[0], g.s[1]);
  return g;
}
wide floor_div(wide a, wide b) { return a / b - (a % b < 0); }
// Rows of one stride s (na from xa, nb from xb): some i, j with xa + i s < xb + j s + wb and xb + j s < xa + i s + wa.
bool lattices_meet(wide xa, wide na, wide wa, wide xb, wide nb, wide wb, wide s) {
  const wide d = xb - xa;
  if (s == 0) return d < wa && -d < wb;
  const wide lo = std::max(floor_div(-wb - d, s) + 1, 1 - na), hi = std::min(-floor_div(d - wa, s) - 1, nb - 1);
  return lo <= hi;
}
}  // namespace

bool rows_apart(const Rows2& r) {
  const Grid2 g = canonical(r, false);
  const wide inner = g.n[1] > 1 ? (g.n[1] - 1) * g.s[1] + g.width : g.width;
  return (g.n[1] == 1 || g.s[1] >= g.width) && (g.n[0] == 1 || g.s[0] >= inner);
}

bool rows_meet(const Rows2& ra, const Rows2& rb) {
  if (ra.n[0] <= 0 || ra.n[1] <= 0 || rb.n[0] <= 0 || rb.n[1] <= 0) return false;
  Grid2 a = canonical(ra, true), b = canonical(rb, true);
  if (a.last() <= b.base || b.last() <= a.base) return false;
  // Cuts of one row: what the inner dimensions span lies apart as a whole.
  if (a.s[0] == b.s[0] || a.n[0] == 1 || b.n[0] == 1) {
    auto span = [](const Grid2& g) { return g.width + (g.n[1] - 1) * g.s[1]; };
    if (!lattices_meet(a.base, a.n[0], span(a), b.base, b.n[0], span(b), std::max(a.s[0], b.s[0]))) return false;
  }
  // the dimension with more rows is looked at as a whole, the other row by row
  auto split = [](const Grid2& g) { return g.n[0] >= g.n[1] ? 0 : 1; };
  const int la = split(a), lb = split(b);
  for (wide i = 0; i < a.n[1 - la]; ++i) {
    const wide xa = a.base + i * a.s[1 - la];
    for (wide j = 0; j < b.n[1 - lb]; ++j) {
      const wide xb = b.base + j * b.s[1 - lb];
      if (xa + a.width + (a.n[la] - 1) * a.s[la] <= xb || xb + b.width + (b.n[lb] - 1) * b.s[lb] <= xa) continue;
      if (a.s[la] == b.s[lb] || a.n[la] == 1 || b.n[lb] == 1) {
        if (lattices_meet(xa, a.n[la], a.width, xb, b.n[lb], b.width, std::max(a.s[la], b.s[lb]))) return true;
      } else if (a.n[la] <= b.n[lb]) {
        for (wide k = 0; k < a.n[la]; ++k)
          if (lattices_meet(xa + k * a.s[la], 1, a.width, xb, b.n[lb], b.width, b.s[lb])) return true;
      } else {
        for (wide k = 0; k < b.n[lb]; ++k)
          if (lattices_meet(xa, a.n[la], a.width, xb + k * b.s[lb], 1, b.width, a.s[la])) return true;
      }
    }
  }
  return false;
}

int launch_check(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(AIB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return AIB_OK;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link-time libcuda dependency)
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

int make_map_3d_u8(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1_bytes,
                   uint64_t s2_bytes, uint32_t b0, uint32_t b1, uint32_t b2) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(AIB_ECUDA, "cuTensorMapEncodeTiled is not available");
  if ((reinterpret_cast<uintptr_t>(base) & 15) || (s1_bytes & 15) || (s2_bytes & 15))
    return fail(AIB_EINVAL, "tensor map: base/strides must be 16-byte aligned");
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {s1_bytes, s2_bytes};
  cuuint32_t box[3] = {b0, b1, b2};
  cuuint32_t es[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIB_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return AIB_OK;
}

int make_map(CUtensorMap* map, CUtensorMapDataType dtype, int elem_bytes, int rank, const void* base,
             const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(AIB_ECUDA, "cuTensorMapEncodeTiled is not available");
  if (rank < 1 || rank > 5) return fail(AIB_EINVAL, "tensor map: rank %d", rank);
  if (reinterpret_cast<uintptr_t>(base) & 15) return fail(AIB_EINVAL, "tensor map: base must be 16-byte aligned");
  for (int i = 0; i + 1 < rank; ++i)
    if (strides_bytes[i] & 15) return fail(AIB_EINVAL, "tensor map: strides must be multiples of 16 bytes");
  if ((box[0] * static_cast<uint32_t>(elem_bytes)) & 15)
    return fail(AIB_EINVAL, "tensor map: the inner box must be a multiple of 16 bytes");
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], es[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    es[i] = 1;
    if (i + 1 < rank) s[i] = strides_bytes[i];
  }
  CUresult r = fn(map, dtype, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(AIB_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return AIB_OK;
}

}  // namespace aib

extern "C" {

int aib_abi_version(void) { return AIB_ABI_VERSION; }

const char* aib_last_error(void) { return aib::t_err; }

void aib_set_pdl(int enabled) { aib::g_pdl = enabled ? 1 : 0; }

int aib_debug_knob(int knob, int value) {
  cudaError_t e = cudaSuccess;
  if (knob == 1) {
    const uint32_t v = value > 0 ? static_cast<uint32_t>(value) : 0u;
    e = cudaMemcpyToSymbol(aib::g_aib_spin_override, &v, sizeof(v));
  } else if (knob == 2) {
    const int v = value ? 1 : 0;
    e = cudaMemcpyToSymbol(aib::g_aib_withhold_copies, &v, sizeof(v));
  } else if (knob == 3) {
    if (value < 0 || value > 2) return aib::fail(AIB_EINVAL, "aib_debug_knob(3): value %d not in 0..2", value);
    aib::attn::g_cluster_sizes = value;
  } else if (knob == 4) {
    if (value != 1 && value != 3 && value != 4) return aib::fail(AIB_EINVAL, "aib_debug_knob(4): value %d", value);
    aib::gemv::g_variant = value;
  } else {
    return aib::fail(AIB_EINVAL, "aib_debug_knob: unknown knob %d", knob);
  }
  if (e != cudaSuccess) return aib::fail(AIB_ECUDA, "aib_debug_knob: %s", cudaGetErrorString(e));
  return AIB_OK;
}

int aib_status_read(int* out, int clear) {
  if (!out) return aib::fail(AIB_EINVAL, "aib_status_read: out is NULL");
  int both[2];
  cudaError_t e = cudaMemcpyFromSymbol(both, aib::g_aib_status, sizeof(both));
  if (e != cudaSuccess) return aib::fail(AIB_ECUDA, "aib_status_read: %s", cudaGetErrorString(e));
  *out = both[0] ? both[0] : both[1];
  if (clear) {
    const int z[2] = {0, 0};
    e = cudaMemcpyToSymbol(aib::g_aib_status, z, sizeof(z));
    if (e != cudaSuccess) return aib::fail(AIB_ECUDA, "aib_status_read(clear): %s", cudaGetErrorString(e));
  }
  return AIB_OK;
}

}  // extern "C"
