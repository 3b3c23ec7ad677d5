// Tokens in and out of the 4-bit cache (cache4.h has its format).
//
// rope_cache4: a step's projected rows [q | k | v] to rotated queries and to their page slots.  HD / 8 lanes take a vector of
// HD entries, lane l the entries 4l .. 4l + 3 of both halves: the pairs (j, j + HD / 2) of the rotation lie in one lane, its four
// codes of either half are two bytes that nobody else writes, and the extremes meet by moves between lanes.  One read of the
// rows, one write of a quarter of them: bound by memory for many rows, by its launch for few.
//
// cache4_rows: the way back, the same lanes of HD / 8 with eight entries in a row each.
//
// The entry next to a border between two codes must get the nearer one, whatever a compiler makes of the arithmetic: bfloat16 rows
// are rotated in 32 bits (as the 16-bit cache's are), rounded, and from there differences of bfloat16 numbers and a correctly
// rounded division leave a border only where entries lie 2^16 apart; 32-bit rows are rotated and divided in 64 bits.
#include "cache4.h"
#include "kvcm_hip.h"

namespace kvcm {
namespace {

constexpr int kThreads = 256;

// Four entries, from any element on.
template <class T> struct Four;
template <> struct Four<bf16_t> {
  typedef uint16_t raw __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ void load(const bf16_t* p, float x[4]) {
    const raw r = *reinterpret_cast<const raw*>(p);
    for (int i = 0; i < 4; ++i) x[i] = bf16_bits_to_float(r[i]);
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float x[4]) {
    raw r;
    for (int i = 0; i < 4; ++i) r[i] = float_to_bf16_bits(x[i]);
    *reinterpret_cast<raw*>(p) = r;
  }
};
template <> struct Four<float> {
  typedef float raw __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ void load(const float* p, float x[4]) {
    const raw r = *reinterpret_cast<const raw*>(p);
    for (int i = 0; i < 4; ++i) x[i] = r[i];
  }
  static __device__ __forceinline__ void store(float* p, const float x[4]) {
    raw r;
    for (int i = 0; i < 4; ++i) r[i] = x[i];
    *reinterpret_cast<raw*>(p) = r;
  }
};

__device__ __forceinline__ void rotate_in(float& a, float& b, float cs, float sn, bf16_t) {
  rotate_pair(a, b, cs, sn);
  a = round_to<bf16_t>(a);
  b = round_to<bf16_t>(b);
}
__device__ __forceinline__ void rotate_in(float& a, float& b, float cs, float sn, float) {
  const double x = a, y = b;      // products of 32-bit numbers are exact in 64 bits
  a = static_cast<float>(x * cs - y * sn);
  b = static_cast<float>(y * cs + x * sn);
}

__device__ __forceinline__ float step_of(float high, float low, bf16_t) { return round_to<bf16_t>((high - low) / 15.0f); }
__device__ __forceinline__ float step_of(float high, float low, float) {
  return round_to<bf16_t>(static_cast<float>((static_cast<double>(high) - low) / 15.0));
}
__device__ __forceinline__ float steps_from(float x, float low, float step, bf16_t) { return rintf((x - low) / step); }
__device__ __forceinline__ float steps_from(float x, float low, float step, float) {
  return static_cast<float>(rint((static_cast<double>(x) - low) / step));
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) rope_cache4_kernel(const T* qkv, int stride, T* q_out, int q_stride, uint8_t* __restrict__ cache,
                                                               const int* __restrict__ slots, const float2* __restrict__ cos_sin, long long vectors, int first,
                                                               int nh, int nkv, int page, unsigned num_slots) {
  constexpr int G = HD / 8;
  const long long at = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / G;
  if (at >= vectors) return;      // all lanes of a vector together
  const int l = threadIdx.x % G, heads = nh + 2 * nkv - first;
  const long long row = at / heads;
  const int head = static_cast<int>(at % heads) + first;      // queries, keys, values
  const bool value = head >= nh + nkv;
  unsigned slot = 0;
  if (head >= nh) {
    slot = static_cast<unsigned>(slots[row]);
    if (slot >= num_slots) return;      // -1: a padding row, nothing to keep
  }
  float x[8];
  const T* src = qkv + row * stride + head * HD;
  Four<T>::load(src + 4 * l, x);
  Four<T>::load(src + HD / 2 + 4 * l, x + 4);
  if (cos_sin != nullptr && !value) {
    const float4* angles = reinterpret_cast<const float4*>(cos_sin + row * (HD / 2) + 4 * l);
    const float4 u = angles[0], v = angles[1];
    rotate_in(x[0], x[4], u.x, u.y, T());
    rotate_in(x[1], x[5], u.z, u.w, T());
    rotate_in(x[2], x[6], v.x, v.y, T());
    rotate_in(x[3], x[7], v.z, v.w, T());
  }
  if (head < nh) {
    T* dst = q_out + row * q_stride + head * HD;
    Four<T>::store(dst + 4 * l, x);
    Four<T>::store(dst + HD / 2 + 4 * l, x + 4);
    return;
  }
  float high = x[0], neg_low = -x[0], not_finite = x[0] * 0.f;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    high = fmaxf(high, x[i]);
    neg_low = fmaxf(neg_low, -x[i]);
    not_finite += x[i] * 0.f;
  }
  high = group_max<G>(high);
  const float low = round_to<bf16_t>(-group_max<G>(neg_low)) + 0.0f;      // (never -0: a vector's bytes are its values')
  const float step = step_of(high, low, T()) + group_sum<G>(not_finite);      // NaN with an Inf or a NaN among the entries
  const bool codes = step > 0.f && step < __builtin_inff();
  uint32_t half[2] = {0, 0};
  if (codes) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      half[i / 4] |= static_cast<uint32_t>(fminf(fmaxf(steps_from(x[i], low, step, T()), 0.f), 15.f)) << (4 * (i % 4));
  }
  const int kvh = (head - nh) % nkv, tiles = page / kTile4;
  const unsigned pg = slot / page, in_page = slot % page;
  uint8_t* tile = cache + ((static_cast<size_t>(pg) * nkv + kvh) * tiles + in_page / kTile4) * tile4_bytes(HD);
  const int t = in_page % kTile4;
  uint8_t* codes_at = tile + (value ? value4_at(HD) : 0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int u = l + h * G;      // entries 4u .. 4u + 3
    if (!value) {
      *reinterpret_cast<uint16_t*>(codes_at + t * (HD / 2) + 2 * u) = half[h];
    } else if constexpr (HD == 32) {
      codes_at[value4_byte<HD>(t, u)] = half[h] & 255;
      codes_at[value4_byte<HD>(t, u) + 4] = half[h] >> 8;
    } else {
      *reinterpret_cast<uint16_t*>(codes_at + value4_byte<HD>(t, u)) = half[h];
    }
  }
  if (l == 0) {
    const float kept = codes || step == 0.f ? step : __builtin_nanf("");
    reinterpret_cast<uint32_t*>(codes_at + 8 * HD)[t] = float_to_bf16_bits(kept) | static_cast<uint32_t>(float_to_bf16_bits(low)) << 16;
  }
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) cache4_rows_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slots, T* __restrict__ k, int k_stride,
                                                               T* __restrict__ v, int v_stride, long long vectors, int nkv, int page, unsigned num_slots) {
  constexpr int G = HD / 8;
  const long long at = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / G;
  if (at >= vectors) return;
  const int l = threadIdx.x % G;
  const long long row = at / (2 * nkv);
  const int kvh = static_cast<int>(at % (2 * nkv)) % nkv;
  const bool value = at % (2 * nkv) >= nkv;
  const unsigned slot = static_cast<unsigned>(slots[row]);
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot < num_slots) {
    const int tiles = page / kTile4, t = slot % kTile4;
    const uint8_t* tile = cache + ((static_cast<size_t>(slot / page) * nkv + kvh) * tiles + slot % page / kTile4) * tile4_bytes(HD) + (value ? value4_at(HD) : 0);
    const uint32_t pair = reinterpret_cast<const uint32_t*>(tile + 8 * HD)[t];
    uint32_t codes;
    if (!value) {
      codes = *reinterpret_cast<const uint32_t*>(tile + t * (HD / 2) + 4 * l);
    } else if constexpr (HD == 32) {
      const uint8_t* b = tile + value4_byte<HD>(t, 2 * l);
      codes = b[0] | b[4] << 8 | b[8] << 16 | static_cast<uint32_t>(b[12]) << 24;
    } else {
      codes = *reinterpret_cast<const uint16_t*>(tile + value4_byte<HD>(t, 2 * l)) | *reinterpret_cast<const uint16_t*>(tile + value4_byte<HD>(t, 2 * l + 1)) << 16;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(step4(pair), static_cast<float>(codes >> (4 * i) & 15u), low4(pair));      // the product is exact
  }
  T* dst = (value ? v + row * v_stride : k + row * k_stride) + kvh * HD + 8 * l;
  Four<T>::store(dst, x);
  Four<T>::store(dst + 4, x + 4);
}

}  // namespace
}  // namespace kvcm

using namespace kvcm;

extern "C" {

int kvcm_cache4_supported(int nh, int nkv, int hd, int page) { return head4(hd) && nkv > 0 && nh > 0 && nh % nkv == 0 && page > 0 && page % kTile4 == 0; }

int kvcm_rope_cache4(const void* qkv, int dtype, int stride, void* q_out, int q_stride, void* cache, const int* slots, const void* cos_sin, int T, int nh, int nkv,
                     int hd, int pages, int page, hipStream_t stream) {
  KVCM_REQUIRE(kvcm_cache4_supported(nh, nkv, hd, page), "rope_cache4: heads %d, kv heads %d, head_dim %d, pages of %d tokens are not taken", nh, nkv, hd, page);
  KVCM_REQUIRE(dtype == kF32 || dtype == kBF16, "rope_cache4: dtype %d", dtype);
  KVCM_REQUIRE(T >= 0 && pages > 0 && static_cast<long long>(pages) * page < (1ll << 31), "rope_cache4: %d rows, %d pages of %d tokens", T, pages, page);
  KVCM_REQUIRE(nh < 65536 && stride >= (nh + 2 * nkv) * hd && (cos_sin == nullptr || q_stride >= nh * hd), "rope_cache4: rows of %d entries, queries of %d", stride, q_stride);
  if (T == 0) return 0;
  KVCM_REQUIRE(qkv != nullptr && cache != nullptr && slots != nullptr && (cos_sin == nullptr || q_out != nullptr), "rope_cache4: null operand");
  const int first = cos_sin != nullptr ? 0 : nh;      // nothing rotates: the queries are not touched
  const long long vectors = static_cast<long long>(T) * (nh + 2 * nkv - first);
  const long long blocks = (vectors * (hd / 8) + kThreads - 1) / kThreads;
  KVCM_REQUIRE(blocks < (1ll << 31), "rope_cache4: %d rows of %d heads are too many for one launch", T, nh + 2 * nkv);
  KVCM_HEAD4(hd, {
    if (dtype == kBF16)
      rope_cache4_kernel<bf16_t, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const bf16_t*>(qkv), stride, static_cast<bf16_t*>(q_out), q_stride,
                                                                      static_cast<uint8_t*>(cache), slots, static_cast<const float2*>(cos_sin), vectors, first,
                                                                      nh, nkv, page, static_cast<unsigned>(pages) * page);
    else
      rope_cache4_kernel<float, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const float*>(qkv), stride, static_cast<float*>(q_out), q_stride,
                                                                     static_cast<uint8_t*>(cache), slots, static_cast<const float2*>(cos_sin), vectors, first,
                                                                     nh, nkv, page, static_cast<unsigned>(pages) * page);
  });
  return launch_status("rope_cache4");
}

int kvcm_cache4_rows(const void* cache, const int* slots, void* k, int k_stride, void* v, int v_stride, int dtype, int n, int nkv, int hd, int pages, int page,
                     hipStream_t stream) {
  KVCM_REQUIRE(kvcm_cache4_supported(nkv, nkv, hd, page), "cache4_rows: kv heads %d, head_dim %d, pages of %d tokens are not taken", nkv, hd, page);
  KVCM_REQUIRE(dtype == kF32 || dtype == kBF16, "cache4_rows: dtype %d", dtype);
  KVCM_REQUIRE(n >= 0 && pages > 0 && static_cast<long long>(pages) * page < (1ll << 31), "cache4_rows: %d tokens, %d pages of %d", n, pages, page);
  KVCM_REQUIRE(k_stride >= nkv * hd && v_stride >= nkv * hd, "cache4_rows: rows of %d and %d entries", k_stride, v_stride);
  if (n == 0) return 0;
  KVCM_REQUIRE(cache != nullptr && slots != nullptr && k != nullptr && v != nullptr, "cache4_rows: null operand");
  const long long vectors = 2ll * n * nkv, blocks = (vectors * (hd / 8) + kThreads - 1) / kThreads;
  KVCM_REQUIRE(blocks < (1ll << 31), "cache4_rows: %d tokens of %d heads are too many for one launch", n, nkv);
  KVCM_HEAD4(hd, {
    if (dtype == kBF16)
      cache4_rows_kernel<bf16_t, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const uint8_t*>(cache), slots, static_cast<bf16_t*>(k), k_stride,
                                                                      static_cast<bf16_t*>(v), v_stride, vectors, nkv, page, static_cast<unsigned>(pages) * page);
    else
      cache4_rows_kernel<float, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const uint8_t*>(cache), slots, static_cast<float*>(k), k_stride,
                                                                     static_cast<float*>(v), v_stride, vectors, nkv, page, static_cast<unsigned>(pages) * page);
  });
  return launch_status("cache4_rows");
}

}  // extern "C"
