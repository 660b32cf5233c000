// A paged key / value cache in 4 or 8 bits: quantisation as tokens are written
// (gko_kv_cache_write) and reading cached sequences back (gko_kv_cache_read).
//
// One row is one token of one kv head: d values x, kept as d codes of `bits` bits and one
// (scale, zero) pair in the element type. With n = 2^bits - 1:
//   zero  = min x                      (a value of the element type, so it is exact)
//   scale = (max x - min x) / n        (rounded UP to the element type, so no code is cut off)
//   code  = rint((x - zero) / scale)   in [0, n]; the code stands for code * scale + zero
// and |x - (code * scale + zero)| <= scale / 2 up to f32 rounding. Rounding the pair to 16 bits
// costs 4 bytes a row instead of 8 and no accuracy beyond the slightly larger scale. A row with
// a NaN, an infinity or a range beyond f32 gets scale 0 and zero NaN: it reads back as NaN, so a
// bad activation stays visible.
//
// Codes are [pages, kv heads, page, d * bits / 8] bytes (4 bits: channel 2i in the low half of
// byte i), pairs [pages, kv heads, page, 2]; the rows of one page and head are contiguous, which
// is what the attention over the cache reads in one bulk copy. Both kernels are bound by memory:
// a row costs 2 d bytes on one side and d * bits / 8 + 4 on the other.
#include "host_common.h"
#include "sm100_ptx.cuh"

namespace gko {
namespace kv {

struct Params {
  const void* k;  // write: new keys / values; unused by the read
  const void* v;
  int64_t k_st, k_sh, v_st, v_sh;
  uint8_t* k_codes;
  uint8_t* v_codes;
  void* k_pairs;
  void* v_pairs;
  int64_t pages, page_size;
  int64_t tokens;  // write: new tokens; read: packed tokens of the destination
  int hkv;
  const int64_t* slots;  // write
  const int32_t* table;  // read
  int64_t table_stride, table_width;
  const int32_t* cu;
  int b;
  void* k_out;
  void* v_out;
  unsigned* status;
};

// -------------------------------------------------------------- packed pairs of the element type
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using P = __nv_bfloat162;
  static constexpr float kFloor = 7.8886090522101181e-31f;  // 2^-100: 1 / scale stays finite
  static __device__ __forceinline__ __nv_bfloat16 up(float x) { return __float2bfloat16_ru(x); }
};
template <>
struct Pair<__half> {
  using P = __half2;
  static constexpr float kFloor = 5.9604644775390625e-8f;  // 2^-24, the smallest f16
  static __device__ __forceinline__ __half up(float x) { return __float2half_ru(x); }
};

template <typename P>
__device__ __forceinline__ P as_pair(uint32_t w) {
  return *reinterpret_cast<P*>(&w);
}
template <typename P>
__device__ __forceinline__ uint32_t as_word(P p) {
  return *reinterpret_cast<uint32_t*>(&p);
}

// -------------------------------------------------------------- write
// kLanes = d / 8 lanes share a row, eight values (16 bytes) each. Minimum and maximum travel
// together as one packed pair (min x, min -x), NaN kept, so a row needs log2(kLanes) shuffles.
template <typename T, int BITS, int kLanes>
__device__ __forceinline__ void quantise_row(const uint4& raw, uint8_t* codes, T* pair, int part, bool store) {
  using P = typename Pair<T>::P;
  constexpr float kTop = BITS == 4 ? 15.f : 255.f;
  const P a = as_pair<P>(raw.x), b = as_pair<P>(raw.y), c = as_pair<P>(raw.z), d = as_pair<P>(raw.w);
  const P lo2 = __hmin2_nan(__hmin2_nan(a, b), __hmin2_nan(c, d));
  const P hi2 = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
  P both;
  both.x = __hmin_nan(lo2.x, lo2.y);
  both.y = __hneg(__hmax_nan(hi2.x, hi2.y));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
    both = __hmin2_nan(both, as_pair<P>(__shfl_xor_sync(0xffffffffu, as_word(both), o)));
  const float low = Cvt<T>::to_f32(both.x), high = -Cvt<T>::to_f32(both.y);
  float scale = Cvt<T>::to_f32(Pair<T>::up((high - low) / kTop));
  scale = fmaxf(scale, Pair<T>::kFloor);
  const bool fine = fabsf(low) < INFINITY && fabsf(high) < INFINITY && scale < INFINITY;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x, y;
    Cvt<T>::unpack(w[i], x, y);
    q[2 * i] = fine ? (uint32_t)fminf(rintf((x - low) / scale), kTop) : 0u;
    q[2 * i + 1] = fine ? (uint32_t)fminf(rintf((y - low) / scale), kTop) : 0u;
  }
  if (!store) return;
  if constexpr (BITS == 4) {
    uint32_t p = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) p |= q[i] << (4 * i);
    reinterpret_cast<uint32_t*>(codes)[part] = p;
  } else {
    reinterpret_cast<uint2*>(codes)[part] =
        make_uint2(q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24);
  }
  if (part == 0) {
    const float s = fine ? scale : 0.f, z = fine ? low : __int_as_float(0x7fc00000);
    *reinterpret_cast<uint32_t*>(pair) = Cvt<T>::pack(s, z);
  }
}

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(256) kv_write_kernel(const Params p) {
  constexpr int kLanes = D / 8;
  constexpr int kRowBytes = D * BITS / 8;
  const int part = threadIdx.x % kLanes;
  const int64_t rows = p.tokens * p.hkv;
  const int64_t groups = (int64_t)gridDim.x * (256 / kLanes);
  const int64_t limit = p.pages * p.page_size;
  // every lane of a warp runs the same number of rounds: the shuffles need all of them
  const int64_t first = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int64_t rounds = (rows + groups - 1) / groups;
  for (int64_t n = 0; n < rounds; ++n) {
    const int64_t r = first + n * groups;
    const bool in = r < rows;
    const int64_t t = in ? r / p.hkv : 0;
    const int h = in ? (int)(r % p.hkv) : 0;
    const int64_t slot = in ? p.slots[t] : -1;
    const bool store = slot >= 0 && slot < limit;
    if (slot >= limit && part == 0 && p.status) atomicOr(p.status, kStatusBadIndex);
    uint4 kx = make_uint4(0, 0, 0, 0), vx = make_uint4(0, 0, 0, 0);
    if (store) {
      kx = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.k) + t * p.k_st + h * p.k_sh + part * 8);
      vx = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.v) + t * p.v_st + h * p.v_sh + part * 8);
    }
    const int64_t row = store ? ((slot / p.page_size) * p.hkv + h) * p.page_size + slot % p.page_size : 0;
    quantise_row<T, BITS, kLanes>(kx, p.k_codes + row * kRowBytes, reinterpret_cast<T*>(p.k_pairs) + row * 2, part,
                                  store);
    quantise_row<T, BITS, kLanes>(vx, p.v_codes + row * kRowBytes, reinterpret_cast<T*>(p.v_pairs) + row * 2, part,
                                  store);
  }
}

// -------------------------------------------------------------- read
// Eight codes -> eight values of the element type. A code (at most 8 bits) times a scale (at
// most 11) is exact in f32, so the value is rounded once in the sum and once to the type.
template <typename T, int BITS>
__device__ __forceinline__ uint4 expand8(uint2 c, float s, float z) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = BITS == 4 ? (c.x >> (4 * i)) & 15u : ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 255u;
    f[i] = fmaf((float)u, s, z);
  }
  return make_uint4(Cvt<T>::pack(f[0], f[1]), Cvt<T>::pack(f[2], f[3]), Cvt<T>::pack(f[4], f[5]),
                    Cvt<T>::pack(f[6], f[7]));
}

template <int BITS>
__device__ __forceinline__ uint2 load_codes8(const uint8_t* row, int part) {
  if constexpr (BITS == 4) return make_uint2(reinterpret_cast<const uint32_t*>(row)[part], 0u);
  return reinterpret_cast<const uint2*>(row)[part];
}

// d / 8 lanes share a token and walk its heads; the token's sequence is found once by bisection.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(256) kv_read_kernel(const Params p) {
  constexpr int kLanes = D / 8;
  constexpr int kRowBytes = D * BITS / 8;
  const int part = threadIdx.x % kLanes;
  const int64_t t = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (t >= p.tokens) return;
  int lo = 0, hi = p.b;  // the first sequence whose end is past t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  if (lo >= p.b || p.cu[lo] > t) return;  // behind the last sequence: left as it is
  const int64_t pos = t - p.cu[lo];
  const int64_t col = pos / p.page_size;
  const int64_t page = col < p.table_width ? p.table[lo * p.table_stride + col] : -1;
  if (page < 0 || page >= p.pages) {
    if (part == 0 && p.status) atomicOr(p.status, kStatusBadIndex);
    return;
  }
  const int64_t row0 = page * p.hkv * p.page_size + pos % p.page_size;
#pragma unroll 4
  for (int h = 0; h < p.hkv; ++h) {
    const int64_t row = row0 + h * p.page_size;
    const uint2 kc = load_codes8<BITS>(p.k_codes + row * kRowBytes, part);
    const uint2 vc = load_codes8<BITS>(p.v_codes + row * kRowBytes, part);
    float ks, kz, vs, vz;
    Cvt<T>::unpack(reinterpret_cast<const uint32_t*>(p.k_pairs)[row], ks, kz);
    Cvt<T>::unpack(reinterpret_cast<const uint32_t*>(p.v_pairs)[row], vs, vz);
    const int64_t at = (t * p.hkv + h) * kLanes + part;
    reinterpret_cast<uint4*>(p.k_out)[at] = expand8<T, BITS>(kc, ks, kz);
    reinterpret_cast<uint4*>(p.v_out)[at] = expand8<T, BITS>(vc, vs, vz);
  }
}

template <typename T, int D, int BITS>
int launch(const Params& p, bool write, cudaStream_t s) {
  const int64_t rows = write ? p.tokens * p.hkv : p.tokens;
  int64_t blocks = (rows + 256 / (D / 8) - 1) / (256 / (D / 8));
  if (write) {
    const int64_t cap = (int64_t)host::sm_count() * 8;
    if (blocks > cap) blocks = cap;
    kv_write_kernel<T, D, BITS><<<(unsigned)blocks, 256, 0, s>>>(p);
  } else {
    kv_read_kernel<T, D, BITS><<<(unsigned)blocks, 256, 0, s>>>(p);
  }
  return host::cuda_check(cudaGetLastError(), write ? "kv cache write launch" : "kv cache read launch");
}

template <typename T>
int dispatch(int d, int bits, const Params& p, bool write, cudaStream_t s) {
  if (d == 64) return bits == 4 ? launch<T, 64, 4>(p, write, s) : launch<T, 64, 8>(p, write, s);
  return bits == 4 ? launch<T, 128, 4>(p, write, s) : launch<T, 128, 8>(p, write, s);
}

int check(const char* what, int dtype, int bits, int64_t tokens, int64_t hkv, int64_t d, int64_t pages,
          int64_t page_size) {
  using host::fail;
  if (dtype != GKO_F16 && dtype != GKO_BF16)
    return fail(GKO_ERR_UNSUPPORTED, "%s supports float16 and bfloat16 only (dtype code %d)", what, dtype);
  if (bits != 4 && bits != 8) return fail(GKO_ERR_UNSUPPORTED, "%s: codes have 4 or 8 bits, got %d", what, bits);
  if (d != 64 && d != 128)
    return fail(GKO_ERR_UNSUPPORTED, "%s supports head dim 64 or 128, got %lld", what, (long long)d);
  if (tokens < 0 || hkv <= 0 || pages < 0) return fail(GKO_ERR_INVALID, "%s: bad sizes", what);
  if (page_size <= 0 || page_size % 16 || page_size > (1 << 20))
    return fail(GKO_ERR_UNSUPPORTED, "%s: the page size must be a multiple of 16 up to 2^20 tokens, got %lld", what,
                (long long)page_size);
  if (tokens >= (1ll << 31) || hkv > 65535 || pages >= (1ll << 31))
    return fail(GKO_ERR_UNSUPPORTED, "%s: sizes out of range", what);
  return GKO_OK;
}

}  // namespace kv
}  // namespace gko

using namespace gko;
using gko::host::fail;

extern "C" int gko_kv_cache_write(int dtype, int bits, int64_t tokens, int64_t hkv, int64_t d, const void* k,
                                  int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                                  const int64_t* slots, void* k_codes, void* v_codes, void* k_pairs, void* v_pairs,
                                  int64_t pages, int64_t page_size, unsigned int* status, void* stream) {
  int rc = kv::check("kv cache write", dtype, bits, tokens, hkv, d, pages, page_size);
  if (rc) return rc;
  if (tokens == 0) return GKO_OK;
  if (!k || !v || !slots || !k_codes || !v_codes || !k_pairs || !v_pairs)
    return fail(GKO_ERR_INVALID, "kv cache write: null pointer argument");
  if (k_st % 8 || k_sh % 8 || v_st % 8 || v_sh % 8)
    return fail(GKO_ERR_UNSUPPORTED, "kv cache write needs token / head strides that are multiples of 8");
  const void* ptrs[6] = {k, v, k_codes, v_codes, k_pairs, v_pairs};
  for (const void* x : ptrs)
    if (!host::aligned16(x)) return fail(GKO_ERR_UNSUPPORTED, "kv cache write needs 16-byte aligned tensors");
  kv::Params p{};
  p.k = k;
  p.v = v;
  p.k_st = k_st;
  p.k_sh = k_sh;
  p.v_st = v_st;
  p.v_sh = v_sh;
  p.k_codes = static_cast<uint8_t*>(k_codes);
  p.v_codes = static_cast<uint8_t*>(v_codes);
  p.k_pairs = k_pairs;
  p.v_pairs = v_pairs;
  p.pages = pages;
  p.page_size = page_size;
  p.tokens = tokens;
  p.hkv = (int)hkv;
  p.slots = slots;
  p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == GKO_BF16 ? kv::dispatch<__nv_bfloat16>((int)d, bits, p, true, s)
                           : kv::dispatch<__half>((int)d, bits, p, true, s);
}

extern "C" int gko_kv_cache_read(int dtype, int bits, int64_t b, int64_t hkv, int64_t d, int64_t tokens,
                                 const void* k_codes, const void* v_codes, const void* k_pairs, const void* v_pairs,
                                 int64_t pages, int64_t page_size, const int32_t* table, int64_t table_stride,
                                 int64_t table_width, const int32_t* cu_seqlens, void* k, void* v,
                                 unsigned int* status, void* stream) {
  int rc = kv::check("kv cache read", dtype, bits, tokens, hkv, d, pages, page_size);
  if (rc) return rc;
  if (b < 0 || b >= (1ll << 31) || table_width < 0 || table_stride < 0)
    return fail(GKO_ERR_INVALID, "kv cache read: bad sizes");
  if (b == 0 || tokens == 0) return GKO_OK;
  if (!k_codes || !v_codes || !k_pairs || !v_pairs || !table || !cu_seqlens || !k || !v)
    return fail(GKO_ERR_INVALID, "kv cache read: null pointer argument");
  const void* ptrs[6] = {k, v, k_codes, v_codes, k_pairs, v_pairs};
  for (const void* x : ptrs)
    if (!host::aligned16(x)) return fail(GKO_ERR_UNSUPPORTED, "kv cache read needs 16-byte aligned tensors");
  kv::Params p{};
  p.k_codes = static_cast<uint8_t*>(const_cast<void*>(k_codes));
  p.v_codes = static_cast<uint8_t*>(const_cast<void*>(v_codes));
  p.k_pairs = const_cast<void*>(k_pairs);
  p.v_pairs = const_cast<void*>(v_pairs);
  p.pages = pages;
  p.page_size = page_size;
  p.tokens = tokens;
  p.hkv = (int)hkv;
  p.table = table;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.cu = cu_seqlens;
  p.b = (int)b;
  p.k_out = k;
  p.v_out = v;
  p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == GKO_BF16 ? kv::dispatch<__nv_bfloat16>((int)d, bits, p, false, s)
                           : kv::dispatch<__half>((int)d, bits, p, false, s);
}
