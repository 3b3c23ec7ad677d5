// Tokens in and out of the 4-bit cache (cache4.h has its format).
//
// rope_cache4: a step's projected rows [q | k | v] to rotated queries and to their page slots.  HD / 16 lanes take a vector of
// HD entries, lane l the entries 8l .. 8l + 7 of both halves: the pairs (j, j + HD / 2) of the rotation lie in one lane, its eight
// codes of either half are bytes that nobody else writes, and the extremes meet by moves between lanes.  One read of the
// rows, one write of a quarter of them: bound by memory for many rows, by its launch for few.  (Two or four heads of a lane in turn, which
// read the row's angles once for them, are slower: 18 and 22 us instead of 16 with 2,048 rows of 48 heads of 128, the rows read back.)
//
// cache4_rows: the way back: HD / 8 lanes take a token's key and value of a kv head, eight entries in a row of each (16 bytes of bfloat16).
//
// The entry next to a border between two codes must get the nearer one, whatever a compiler makes of the arithmetic: bfloat16 rows
// are rotated in 32 bits (as the 16-bit cache's are), rounded, and from there differences of bfloat16 numbers and a correctly
// rounded division leave a border only where entries lie 2^16 apart; 32-bit rows are rotated and divided in 64 bits.
#include "cache4.h"
#include "kvcm_hip.h"

namespace kvcm {
namespace {

constexpr int kThreads = 256;

// Eight entries, from any element on.
template <class T> struct Eight;
template <> struct Eight<bf16_t> {
  typedef uint16_t raw __attribute__((ext_vector_type(8), aligned(2)));
  static __device__ __forceinline__ void load(const bf16_t* p, float x[8]) {
    const raw r = *reinterpret_cast<const raw*>(p);
    for (int i = 0; i < 8; ++i) x[i] = bf16_bits_to_float(r[i]);
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float x[8]) {
    raw r;
    for (int i = 0; i < 8; ++i) r[i] = float_to_bf16_bits(x[i]);
    *reinterpret_cast<raw*>(p) = r;
  }
};
template <> struct Eight<float> {
  typedef float raw __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ void load(const float* p, float x[8]) {
    const raw a = reinterpret_cast<const raw*>(p)[0], b = reinterpret_cast<const raw*>(p)[1];
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
  }
  static __device__ __forceinline__ void store(float* p, const float x[8]) {
    reinterpret_cast<raw*>(p)[0] = raw{x[0], x[1], x[2], x[3]};
    reinterpret_cast<raw*>(p)[1] = raw{x[4], x[5], x[6], x[7]};
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
  return high - low < __builtin_inff() ? round_to<bf16_t>(static_cast<float>((static_cast<double>(high) - low) / 15.0)) : __builtin_inff();
}
__device__ __forceinline__ float steps_from(float x, float low, float step, bf16_t) { return rintf((x - low) / step); }
__device__ __forceinline__ float steps_from(float x, float low, float step, float) {
  return static_cast<float>(rint((static_cast<double>(x) - low) / step));
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) rope_cache4_kernel(const T* qkv, int stride, T* q_out, int q_stride, uint8_t* __restrict__ cache,
                                                               const int* __restrict__ slots, const float2* __restrict__ cos_sin, int vectors, Divisor heads, int first,
                                                               int nh, int nkv, Divisor page_tiles, unsigned num_slots) {
  constexpr int G = HD / 16;
  const int at = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (at >= vectors) return;      // all lanes of a vector together
  const int l = threadIdx.x % G, row = quotient(at, heads), head = at - row * heads.d + first;      // queries, keys, values
  const bool value = head >= nh + nkv, turns = cos_sin != nullptr && !value;
  // everything that is read is asked for before any of it is looked at
  const unsigned slot = head >= nh ? static_cast<unsigned>(slots[row]) : 0u;
  float4 angles[4] = {};
  if (turns) {
    const float4* from = reinterpret_cast<const float4*>(cos_sin + static_cast<size_t>(row) * (HD / 2) + 8 * l);
#pragma unroll
    for (int i = 0; i < 4; ++i) angles[i] = from[i];
  }
  float x[16];
  const T* src = qkv + static_cast<size_t>(row) * stride + head * HD + 8 * l;
  Eight<T>::load(src, x);
  Eight<T>::load(src + HD / 2, x + 8);
  if (turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rotate_in(x[2 * i], x[8 + 2 * i], angles[i].x, angles[i].y, T());
      rotate_in(x[2 * i + 1], x[9 + 2 * i], angles[i].z, angles[i].w, T());
    }
  }
  if (head < nh) {
    T* dst = q_out + static_cast<size_t>(row) * q_stride + head * HD + 8 * l;
    Eight<T>::store(dst, x);
    Eight<T>::store(dst + HD / 2, x + 8);
    return;
  }
  if (slot >= num_slots) return;      // -1: a padding row, nothing to keep
  float high = x[0], neg_low = -x[0], not_finite = x[0] * 0.f;
#pragma unroll
  for (int i = 1; i < 16; ++i) {
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
    for (int i = 0; i < 16; ++i)
      half[i / 8] |= static_cast<uint32_t>(fminf(fmaxf(steps_from(x[i], low, step, T()), 0.f), 15.f)) << (4 * (i % 8));
  }
  const int kvh = value ? head - nh - nkv : head - nh;
  const int tile = slot / kTile4, t = slot % kTile4, pg = quotient(tile, page_tiles), in_page = tile - pg * page_tiles.d;
  uint8_t* codes_at = cache + ((static_cast<size_t>(pg) * nkv + kvh) * page_tiles.d + in_page) * tile4_bytes(HD) + (value ? value4_at(HD) : 0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int u = 2 * (l + h * G);      // entries 4u .. 4u + 7
    if (!value) {
      *reinterpret_cast<uint32_t*>(codes_at + t * (HD / 2) + 2 * u) = half[h];
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t four = half[h] >> (16 * e) & 0xFFFFu;
        uint8_t* to = codes_at + value4_byte<HD>(t, u + e);
        if constexpr (HD == 32) {
          to[0] = four & 255;
          to[4] = four >> 8;
        } else {
          *reinterpret_cast<uint16_t*>(to) = four;
        }
      }
    }
  }
  if (l == 0) {
    const float kept = codes || step <= 0.f ? fmaxf(step, 0.f) : __builtin_nanf("");      // (a low rounded above the highest entry: no range)
    reinterpret_cast<uint32_t*>(codes_at + 8 * HD)[t] = float_to_bf16_bits(kept) | static_cast<uint32_t>(float_to_bf16_bits(low)) << 16;
  }
}

template <class T, int HD>
__global__ void __launch_bounds__(kThreads) cache4_rows_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slots, T* __restrict__ k, int k_stride,
                                                               T* __restrict__ v, int v_stride, int vectors, Divisor nkv, Divisor page_tiles, unsigned num_slots) {
  constexpr int G = HD / 8;
  const int at = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (at >= vectors) return;
  const int l = threadIdx.x % G, row = quotient(at, nkv), kvh = at - row * nkv.d;
  const unsigned slot = static_cast<unsigned>(slots[row]);
  float x[8] = {}, y[8] = {};
  if (slot < num_slots) {
    const int tile = slot / kTile4, t = slot % kTile4, pg = quotient(tile, page_tiles), in_page = tile - pg * page_tiles.d;
    const uint8_t* keys = cache + ((static_cast<size_t>(pg) * nkv.d + kvh) * page_tiles.d + in_page) * tile4_bytes(HD);
    const uint8_t* values = keys + value4_at(HD);
    const uint32_t key = *reinterpret_cast<const uint32_t*>(keys + t * (HD / 2) + 4 * l);
    uint32_t value;
    if constexpr (HD == 32) {
      const uint8_t* b = values + value4_byte<HD>(t, 2 * l);
      value = b[0] | b[4] << 8 | b[8] << 16 | static_cast<uint32_t>(b[12]) << 24;
    } else {
      value = *reinterpret_cast<const uint16_t*>(values + value4_byte<HD>(t, 2 * l)) | *reinterpret_cast<const uint16_t*>(values + value4_byte<HD>(t, 2 * l + 1)) << 16;
    }
    const uint32_t of_key = reinterpret_cast<const uint32_t*>(keys + 8 * HD)[t], of_value = reinterpret_cast<const uint32_t*>(values + 8 * HD)[t];
#pragma unroll
    for (int i = 0; i < 8; ++i) {      // (the products are exact)
      x[i] = fmaf(step4(of_key), static_cast<float>(key >> (4 * i) & 15u), low4(of_key));
      y[i] = fmaf(step4(of_value), static_cast<float>(value >> (4 * i) & 15u), low4(of_value));
    }
  }
  Eight<T>::store(k + static_cast<size_t>(row) * k_stride + kvh * HD + 8 * l, x);
  Eight<T>::store(v + static_cast<size_t>(row) * v_stride + kvh * HD + 8 * l, y);
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
  const int first = cos_sin != nullptr ? 0 : nh, heads = nh + 2 * nkv - first;      // nothing rotates: the queries are not touched
  const long long vectors = static_cast<long long>(T) * heads, blocks = (vectors * (hd / 16) + kThreads - 1) / kThreads;
  // (quotients below 2^30, 2^32 threads of a launch)
  KVCM_REQUIRE(vectors < (1ll << 30) && blocks < (1ll << 24), "rope_cache4: %d rows of %d heads are too many for one launch", T, nh + 2 * nkv);
  KVCM_HEAD4(hd, {
    const auto go = [&](auto t) {
      using E = decltype(t);
      rope_cache4_kernel<E, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const E*>(qkv), stride, static_cast<E*>(q_out), q_stride, static_cast<uint8_t*>(cache), slots,
                                                                 static_cast<const float2*>(cos_sin), static_cast<int>(vectors), divisor(heads), first, nh, nkv,
                                                                 divisor(page / kTile4), static_cast<unsigned>(pages) * page);
    };
    if (dtype == kBF16) go(bf16_t());
    else go(float());
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
  const long long vectors = static_cast<long long>(n) * nkv, blocks = (vectors * (hd / 8) + kThreads - 1) / kThreads;
  KVCM_REQUIRE(vectors < (1ll << 30) && blocks < (1ll << 24), "cache4_rows: %d tokens of %d heads are too many for one launch", n, nkv);
  KVCM_HEAD4(hd, {
    const auto go = [&](auto t) {
      using E = decltype(t);
      cache4_rows_kernel<E, HD><<<blocks, kThreads, 0, stream>>>(static_cast<const uint8_t*>(cache), slots, static_cast<E*>(k), k_stride, static_cast<E*>(v), v_stride,
                                                                 static_cast<int>(vectors), divisor(nkv), divisor(page / kTile4), static_cast<unsigned>(pages) * page);
    };
    if (dtype == kBF16) go(bf16_t());
    else go(float());
  });
  return launch_status("cache4_rows");
}

}  // extern "C"
