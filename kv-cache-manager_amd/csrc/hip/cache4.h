// The paged cache held in 4 bits: what its bytes mean.
//
// Of each token and kv head, of the key and of the value, a vector x of hd entries is kept as
//   low = bf16(min x),  step = bf16((max x - low) / 15),  code = rint((x - low) / step) in 0..15  (0 where step is 0)
// and stands for low + step * code: off by at most step / 2 from low on (rounding step to bfloat16 moves the highest entry by up to
// 15 * 2^-8 of a step, which is less).  A vector of bfloat16 has nothing below low; one of float can, where low was rounded up, and
// what lies there is off by up to 2^-8 |min x|, however small a step is.  A vector with an Inf or a NaN (or whose range passes the
// largest float) has step = NaN and reads as NaN in all its places; its codes are 0.
//
// The cache is bytes [pages][kv heads][page / 16][16 * (hd + 8)]: tiles of 16 tokens, one behind the other, each
//   key codes       8 * hd bytes   token t's at t * hd / 2; entry d in byte d / 2, the even one in its low half
//   key pairs       64 bytes       step | low << 16 of each token
//   value codes     8 * hd bytes   in words of 4 entries of two neighbouring tokens (below)
//   value pairs     64 bytes
// so that a tile is one piece of memory (2,176 bytes at hd 128) and everything in it is aligned to 16 bytes.
//
// The two products of attention want their operands packed along the axis they add over: keys along entries, as they lie;
// values along tokens, while they arrive a token at a time.  A word of value codes therefore holds entries 4u .. 4u + 3 of the
// tokens 2p (low half) and 2p + 1 (high half): (word >> 4s) & 0x000F000F are the codes of entry 4u + s of both tokens side by
// side, the pair a matrix operand wants, and a token's half word is written by nobody else.  Sixteen chunks of C = hd / 16
// entries follow one another inside a group of four tokens, so that lane c of 16 reads its C entries of four tokens as C / 2
// words in a row.  (hd 32, C = 2: a byte holds two entries of a token, the bytes of a word are tokens 0, 2, 1, 3.)
#pragma once
#include "common.h"

namespace kvcm {

constexpr int kTile4 = 16;
constexpr int tile4_bytes(int hd) { return kTile4 * (hd + 8); }
constexpr int value4_at(int hd) { return 8 * hd + 64; }      // of the value codes in a tile

// Byte, in a tile's value codes, of the four entries 4u .. 4u + 3 of token t (two bytes; hd 32: of entries 4u, 4u + 1, and 4 on of 4u + 2, 4u + 3).
template <int HD>
__device__ __forceinline__ int value4_byte(int t, int u) {
  constexpr int C = HD / 16;
  const int four = t / 4, pair = t / 2 % 2, odd = t % 2;
  if constexpr (C == 2) return 4 * (four * 16 + 2 * u) + 2 * odd + pair;
  else return 4 * ((four * 16 + 4 * u / C) * (C / 2) + pair * (C / 4) + u % (C / 4)) + 2 * odd;
}

__device__ __forceinline__ float step4(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float low4(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }

// Division by a number that the host knows: these kernels are a few microseconds long, and dividing by a variable takes some twenty
// instructions each time.  n / d = 2 n * by / 2^32 / 2^shift with by = 2^(31 + shift) / d rounded up, shift = log2 d rounded down: too much
// by less than n / 2^(31 + shift) * d / d, below 1 / d for n < 2^30.
struct Divisor {
  int d, shift;
  unsigned by;
};
inline Divisor divisor(int d) {
  const int shift = 31 - __builtin_clz(d);
  return Divisor{d, shift, static_cast<unsigned>(((1ull << (31 + shift)) + d - 1) / d)};
}
__device__ __forceinline__ int quotient(int n, const Divisor& d) { return static_cast<int>(__umulhi(2u * n, d.by) >> d.shift); }

inline bool head4(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

}  // namespace kvcm

// Runs `...` with HD a constant.
#define KVCM_HEAD4(hd, ...)                                                       \
  switch (hd) {                                                                   \
    case 32: { constexpr int HD = 32; __VA_ARGS__; break; }                       \
    case 64: { constexpr int HD = 64; __VA_ARGS__; break; }                       \
    case 128: { constexpr int HD = 128; __VA_ARGS__; break; }                     \
    default: { constexpr int HD = 256; __VA_ARGS__; }                             \
  }
