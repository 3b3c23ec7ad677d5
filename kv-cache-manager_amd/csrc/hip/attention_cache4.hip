// Attention over the 4-bit cache (cache4.h): softmax(scale * q . k) v over a row's visible tokens, max(0, p + 1 - window) <= t <= p,
// for rows of different sequences and for runs of consecutive positions.
//
// The heads that share a kv head read the same keys: the rows of a walk are (position, head of the group) pairs, position by
// position, 16 of them to a tile, RT tiles to a wave.  A single token of a sequence is a run of one.  A wave walks its tokens 32 at a
// time with a running maximum m, on the matrix cores (16x16x32, bfloat16), both products transposed:
//   S^T[token][row] = K[token][entry] Q^T[entry][row],   O^T[entry][row] += V^T[entry][token] P^T[token][row]
// so that the scores of a lane all belong to one row (lane % 16) and are, as they stand, what the second product takes from that
// lane.  Nothing passes through LDS.
//
// Codes become operands without arithmetic: in bfloat16 0x4180 | c << 3 is B + c with B = 16, exactly, and one shift and one bit operation
// give two of them (8 instructions for 8 codes; keys and values both lie in the order that this needs).  0x4300 | c, 128 + c, spares one of
// the eight, 1 to 3 % of the time (6 % of prompts with 256 entries), but sums 5 times as large lose as much more of their 32 bits: with keys
// and queries of 20 +- 20 a score was off by up to 0.06 at 128 entries and 0.1 at 256, and is by 0.005 and 0.008.  With f the scale times
// log2 e,
//   f q . k - m = (f step) (q . (B + c)) + [low (f sum q) - B step (f sum q) - m]
// where the bracket is a matrix instruction of its own, m its accumulator's start: a pair (step, low) as it lies in the cache is an
// operand, against f sum q as three bfloat16 numbers (24 bits) and -B times them.  (Float rows and 128 entries or more: q . (B + c) starts
// from -(B + 8) sum q, with the small terms of float queries before the large, and 8 step is in the bracket: sums stay nearer to what they
// come to.)  One multiplication and addition for each score leaves the exponential's argument.
//   sum p v = sum (p step) (B + c) - (B + 8) sum (p step) + sum p (low + 8 step)
// where p step is the operand: as a sum of bfloat16 numbers, two for single tokens (16 bits, as attention_decode keeps of p), one for runs (as
// attention_prefill rounds p), three for float rows (which keep all 24 bits, as q does).  With normal keys and values, 1,000 tokens of 128 entries, one number
// leaves the output off by 2.3e-3 of its norm, of which rounding the output itself is 1.65e-3, and two by 1.65e-3.  The second costs single tokens 2 to 8 %
// (eight rows of 32,768 tokens 51.9 and 55.6 us), with more than 16 heads to a kv head 4 to 15 (32 over one of 64, 1,500 rows of 400 18.4 and 21.2),
// and would cost runs 14 to 30 (a prompt of 2,048 42.0 and 54.6 us).  The sum of p step comes from one more matrix instruction with ones, so that
// B + 8 cancels exactly as rounded; what the rounding is multiplied with is c - 8, as far from 0 as the values are from their middle.  sum p and
// sum p (low + 8 step) stay in 32 bits.
//
// m is not the largest score but one that no score passes by more than 2^6: it moves in few chunks, and only then do a row's four lanes
// compare what they have and the sums get scaled.
//
// How the work is laid out (a rule on sizes, `plan`): the W waves of a workgroup share a tile of rows and take every W-th 32 tokens; their m, l, o
// meet in LDS.  Single tokens are bound by reading the cache, runs of many rows by vector instructions (some 270 of a wave for 32 rows and 32
// tokens of 128 entries, beside 38 matrix instructions).  Waves with rows of their own walk four times as long, and the last of them
// alone: 446 us instead of 285 for portions of prompts behind contexts of 3,000 to 8,000 tokens (32 heads over 8 of 128); with operands that four such
// waves make for one another in LDS, a quarter fewer instructions and a barrier every 64 tokens, 475 us.
// Contexts are cut into segments that run as workgroups of their own while there are few; a second launch joins what they leave
// in scratch (o, m, l in 32 bits, in the order of the segments).

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "cache4.h"
#include "kvcm_hip.h"

namespace kvcm {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kChunk = 32;      // tokens a wave takes at a time: two tiles of the cache
constexpr float kAhead = 6.f;   // m follows when a score is 2^6 ahead of it

__device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2)); }
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// B + c of the codes 4s .. 4s + 3 bits into either half of a word: one bit operation takes the mask and B, where one of them lies in a vector
// register (`mask`; an instruction reads one scalar register).
constexpr int B = 16;
constexpr uint32_t kMask = 0x00780078u;
__device__ __forceinline__ uint32_t codes(uint32_t word, int s, uint32_t mask) { return ((s == 0 ? word << 3 : word >> (4 * s - 3)) & mask) | 0x41804180u; }

// The low halves of two words side by side, and the high ones.
__device__ __forceinline__ uint32_t pick_low(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pick_high(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Numbers as sums of bfloat16 ones: queries one for rows of bfloat16, three for float (24 bits); p step (NP of the kernel) so many, or two for
// single tokens of bfloat16.
template <class T> constexpr int kTerms = 1;
template <> constexpr int kTerms<float> = 3;
// Whether the sum over a key's codes starts from -(B + 8) sum q.  Bfloat16 rows of fewer than 128 entries have shorter sums and need the start's
// registers more (64 entries, a prompt of 2,048: two waves to a SIMD instead of three, 48.7 us and 41.9; 128 entries: 63.6 and 63.7).
template <class T, int HD> constexpr bool kFromMiddle = kTerms<T> > 1 || HD >= 128;

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * i);
      w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
    }
  }
}

// What a lane holds of 32 tokens: of either tile, a key's HD / 4 codes, four tokens' HD / 16 value codes, and the pairs of
// these four.
template <int HD>
struct Chunk {
  uint32_t k[2][HD / 32], v[2][HD / 32];
  u32x4 kp[2], vp[2];
  uint32_t of_token[2];      // the pair of token lane % 16's key
};

// Where rows come from: single tokens (where = row_seq, lens = ctx_lens) or runs (run_start, seq_start).
struct Rows {
  const int *where, *lens;
  int seqs, total;      // sequences with a table; rows
  bool runs;
};

struct Shape {
  int q_stride, out_stride, table_stride, nh, pages, max_segs, tiles;
  Divisor nkv, group, segs, page_tiles, segment;      // segment: in chunks (and max_segs 1: not looked at)
  float scale_log2;
  int window, max_context, tile_rows;
};

struct Span {
  int row0, rows, seq, ctx0;      // first row, (position, head) pairs, sequence, context of the first row less one
};

// The run that unit (token or sequence) `unit` walks for; rows is 0 where there is none.
__device__ __forceinline__ Span span_of(const Rows& r, const Shape& s, int unit) {
  if (!r.runs) {
    const int seq = r.where[unit];
    return Span{unit, s.group.d, seq, static_cast<unsigned>(seq) < static_cast<unsigned>(r.seqs) ? max(0, r.lens[unit]) - 1 : -1};
  }
  const int a = max(0, r.where[unit]), b = min(r.total, r.where[unit + 1]);
  return Span{a, max(0, b - a) * s.group.d, unit, min(r.lens[unit], 0x7FFFFFFF - r.total)};
}
// Tokens that position i of a span sees: [first, end).
__device__ __forceinline__ int end_of(const Span& p, const Shape& s, int i) { return max(0, min(p.ctx0 + i + 1, s.max_context)); }
__device__ __forceinline__ int first_of(const Span& p, const Shape& s, int i) {
  const int end = end_of(p, s, i), ctx = p.ctx0 + i + 1;      // (below 0 for a run that begins in front of its sequence)
  return s.window > 0 && ctx > s.window ? min(end, ctx - s.window) : 0;
}

// Which segments the tokens of a tile of rows lie in.
struct Cut {
  int first, segs;
};
__device__ __forceinline__ Cut cut_of(const Span& p, const Shape& s, int block_first, int block_last) {
  if (s.max_segs == 1) return Cut{0, 1};
  const int lo = first_of(p, s, quotient(block_first, s.group)), hi = end_of(p, s, quotient(block_last, s.group));
  const int first = quotient(lo / kChunk, s.segment);
  return Cut{first, hi > lo ? quotient((hi - 1) / kChunk, s.segment) - first + 1 : 1};
}

__device__ __forceinline__ void load_eight(const float* p, float x[8]) {
  typedef float raw __attribute__((ext_vector_type(4), aligned(4)));
  const raw a = reinterpret_cast<const raw*>(p)[0], b = reinterpret_cast<const raw*>(p)[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
}
template <class T, int N>
__device__ __forceinline__ void store_some(T* p, const float (&x)[N]) {
  if constexpr (sizeof(T) == 2) {
    typedef uint16_t raw __attribute__((ext_vector_type(N), aligned(2)));
    raw r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = float_to_bf16_bits(x[i]);
    *reinterpret_cast<raw*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = x[i];
  }
}

__device__ __forceinline__ uint32_t in_vector_register(uint32_t x) {
  uint32_t r;
  asm("v_mov_b32 %0, %1" : "=v"(r) : "s"(x));
  return r;
}

// blockIdx.x: kv head (fastest: with eight of them each of the chip's eight parts keeps to one), then segment, then tile of rows, the last
// tile first (it sees the most keys); blockIdx.y: token or sequence.
// Waves on a SIMD that the registers are bounded for.  (Two tiles of rows and 64 entries: three, also where single tokens' second term of p step then
// spills two or three registers: 32 heads over one, 1,500 rows of 400 tokens 21.2 us, with two waves 27.8; 2,000 of 40 12.7 and 12.0.)
constexpr int least_waves(bool wide, int hd, int rt) {
  return hd == 256 ? 1 : wide || (rt == 2 && hd == 128) ? 2 : rt == 2 || hd == 128 ? 3 : 4;
}
template <class T, int HD, int RT, int W, int NP>
__global__ void __launch_bounds__(W * kWave, least_waves(sizeof(T) == 4, HD, RT)) attention4_kernel(const T* __restrict__ q, T* __restrict__ out, const uint8_t* __restrict__ cache,
                                                              const int* __restrict__ tables, Rows rows, Shape sh, float* __restrict__ scratch) {
  constexpr int KS = HD / 32, C = HD / 16, NT = kTerms<T>;
  constexpr bool MID = kFromMiddle<T, HD>;
  const int rest = quotient(blockIdx.x, sh.nkv), kvh = blockIdx.x - rest * sh.nkv.d, tile_up = quotient(rest, sh.segs), part = rest - tile_up * sh.max_segs;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, n16 = lane % 16, kq = lane / 16;
  const int group = sh.group.d;
  const Span span = span_of(rows, sh, blockIdx.y);
  const int first = (sh.tiles - 1 - tile_up) * sh.tile_rows;      // of the span's pairs
  if (first >= span.rows) return;
  const int last = min(first + sh.tile_rows, span.rows) - 1;
  // the workgroup's tokens, and the segment of them that it takes
  const Cut cut = cut_of(span, sh, first, last);
  const int segs = cut.segs;
  if (part >= segs) return;
  const int seg_first = sh.max_segs == 1 ? 0 : (cut.first + part) * sh.segment.d * kChunk;
  const int seg_end = sh.max_segs == 1 ? 0x7FFFFFFF : static_cast<int>(min(0x7FFFFFFFu, static_cast<unsigned>(seg_first) + sh.segment.d * kChunk));
  const int at_first = quotient(first, sh.group), at_last = quotient(last, sh.group);
  const int lo = max(first_of(span, sh, at_first), seg_first), hi = min(end_of(span, sh, at_last), seg_end);
  const int all_lo = first_of(span, sh, at_last), all_hi = end_of(span, sh, at_first);      // what every row sees

  const u32x4 ones{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  int row_lo[RT], row_hi[RT];
  u32x4 qf[RT][NT][KS], q_sum[RT];
  f32x4 start[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int f = min(first + 16 * rt + n16, span.rows - 1);      // pairs past the end repeat the last one; they are never stored
    const int at = quotient(f, sh.group), head = kvh * group + f - at * group;
    row_lo[rt] = max(first_of(span, sh, at), seg_first);
    row_hi[rt] = min(end_of(span, sh, at), seg_end);
#pragma unroll
    for (int c = 0; c < KS; ++c) {      // codes come in the order 0 4 1 5 2 6 3 7
      const T* from = q + static_cast<size_t>(span.row0 + at) * sh.q_stride + head * HD + kq * (HD / 4) + 8 * c;
      if constexpr (NT == 1) {
        typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
        const raw x = *reinterpret_cast<const raw*>(from);
        qf[rt][0][c] = u32x4{pick_low(x[0], x[2]), pick_high(x[0], x[2]), pick_low(x[1], x[3]), pick_high(x[1], x[3])};
      } else {
        float x[8];
        load_eight(from, x);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qf[rt][n][c][i] = pack(x[i], x[i + 4]);
            x[i] -= bf16_bits_to_float(qf[rt][n][c][i] & 0xFFFFu);
            x[i + 4] -= bf16_bits_to_float(qf[rt][n][c][i] >> 16);
          }
      }
    }
    f32x4 sums{0.f, 0.f, 0.f, 0.f};      // each of them the row's
#pragma unroll
    for (int n = NT - 1; n >= 0; --n)
#pragma unroll
      for (int c = 0; c < KS; ++c) sums = product(ones, qf[rt][n][c], sums);
    const float sum = sums[0];
    const float less = -(B + 8.f) * sum;
    start[rt] = f32x4{less, less, less, less};
    // against a pair (step, low), three times: what step and low are multiplied with (the first lane of a row; the others' is 0)
    float left = kq == 0 ? sum * sh.scale_log2 : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float term = i < 3 ? round_to<bf16_t>(left) : 0.f;
      q_sum[rt][i] = pack((MID ? 8.f : -B) * term, term);
      left -= term;
    }
  }

  float limit[RT], l[RT], of_mid[RT];      // limit: how far ahead of m a score may be (-FLT_MAX: no score yet, and m is 0)
  f32x4 less_m[RT], o[RT][C], of_step[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    limit[rt] = -FLT_MAX;
    l[rt] = of_mid[rt] = 0.f;
    less_m[rt] = of_step[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < C; ++d) o[rt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int chunk_first = lo / kChunk + wave, chunk_end = (static_cast<unsigned>(hi) + kChunk - 1) / kChunk;      // every W-th of them
  const int* table = tables + static_cast<size_t>(max(span.seq, 0)) * sh.table_stride;      // (looked at only where there are tokens)
  const int k_at = n16 * (HD / 2) + kq * (HD / 8), v_at = value4_at(HD) + (kq * 16 + n16) * (HD / 8);
  const int kp_at = 8 * HD + kq * 16, vp_at = value4_at(HD) + 8 * HD + kq * 16, token_at = 8 * HD + n16 * 4;
  const uint32_t mask = in_vector_register(kMask);

  // Of either tile of a chunk: where it lies, and whether it has tokens.  One past the end stands for the last, one whose page is none for
  // the cache's first page (nobody looks at their tokens): no load and no address is behind a branch.
  struct Ids {
    size_t at[2];
    bool some[2];
  };
  const int tile_end = (hi + kTile4 - 1) / kTile4;
  auto ids_of = [&](int chunk) {
    Ids r;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int tile = min(2 * chunk + j, tile_end - 1), p = quotient(tile, sh.page_tiles), page = table[p];
      r.some[j] = 2 * chunk + j < tile_end && static_cast<unsigned>(page) < static_cast<unsigned>(sh.pages);
      const unsigned of_cache = static_cast<unsigned>(page) < static_cast<unsigned>(sh.pages) ? page : 0;
      r.at[j] = ((static_cast<size_t>(of_cache) * sh.nkv.d + kvh) * sh.page_tiles.d + (tile - p * sh.page_tiles.d)) * tile4_bytes(HD);
    }
    return r;
  };
  auto request_keys = [&](const Ids& ids, Chunk<HD>& c) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* p = cache + ids.at[j];
      load_words(p + k_at, c.k[j]);
      c.kp[j] = *reinterpret_cast<const u32x4*>(p + kp_at);
      c.of_token[j] = *reinterpret_cast<const uint32_t*>(p + token_at);
    }
  };
  auto request_values = [&](const Ids& ids, Chunk<HD>& c) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* p = cache + ids.at[j];
      load_words(p + v_at, c.v[j]);
      c.vp[j] = *reinterpret_cast<const u32x4*>(p + vp_at);
    }
  };

  // s = scale * log2 e * q . k - m
  auto score = [&](const Chunk<HD>& c, f32x4 (&s)[RT][2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 kf[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[k] = u32x4{codes(c.k[j][k], 0, mask), codes(c.k[j][k], 1, mask), codes(c.k[j][k], 2, mask), codes(c.k[j][k], 3, mask)};
      const u32x4 pairs{c.of_token[j], c.of_token[j], c.of_token[j], c.of_token[j]};
      float step[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) step[i] = step4(c.kp[j][i]) * sh.scale_log2;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const f32x4 rest = product(pairs, q_sum[rt], less_m[rt]);
        f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = NT - 1; n > 0; --n)
#pragma unroll
          for (int k = 0; k < KS; ++k) x = product(kf[k], qf[rt][n][k], x);
        if constexpr (NT > 1) x += start[rt];
        else if constexpr (MID) x = start[rt];
#pragma unroll
        for (int k = 0; k < KS; ++k) x = product(kf[k], qf[rt][0][k], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[rt][j][i] = fmaf(step[i], x[i], rest[i]);
      }
    }
  };
  // WHOLE: every row sees all 32 tokens
  auto add = [&](auto whole, int chunk, const Ids& ids, const Chunk<HD>& c, f32x4 (&s)[RT][2]) {
    constexpr bool WHOLE = decltype(whole)::value;
    bool ok[RT][2][4];
    float top[RT];
    bool move = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = -FLT_MAX;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = chunk * kChunk + 16 * j + 4 * kq + i;
          ok[rt][j][i] = WHOLE || ((t >= row_lo[rt]) & (t < row_hi[rt]) & ids.some[j]);
          s[rt][j][i] = ok[rt][j][i] ? s[rt][j][i] : -FLT_MAX;
          top[rt] = fmaxf(top[rt], s[rt][j][i]);
        }
      move |= top[rt] > limit[rt];
    }
    if (__builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float most = rows_max(top[rt]);
        const bool moves = most > limit[rt];
        const float by = moves ? most : 0.f, alpha = limit[rt] == -FLT_MAX ? 1.f : __builtin_amdgcn_exp2f(-by);      // (no score yet: nothing to scale)
        limit[rt] = moves ? kAhead : limit[rt];
        less_m[rt] -= by;
        l[rt] *= alpha;
        of_mid[rt] *= alpha;
        of_step[rt] *= alpha;
#pragma unroll
        for (int d = 0; d < C; ++d) o[rt][d] *= alpha;
#pragma unroll
        for (int j = 0; j < 2; ++j) s[rt][j] -= by;
      }
    }
    u32x4 pf[RT][NP];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float p_step[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // zero times what a place that is not seen holds (an Inf, a NaN) would not be zero
          const uint32_t pair = ok[rt][j][i] ? c.vp[j][i] : 0u;
          const float e = __builtin_amdgcn_exp2f(s[rt][j][i]), p = ok[rt][j][i] ? e : 0.f, step = step4(pair);
          l[rt] += p;
          of_mid[rt] = fmaf(p, fmaf(8.f, step, low4(pair)), of_mid[rt]);
          p_step[j][i] = p * step;
        }
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t two = pack(p_step[j][2 * i], p_step[j][2 * i + 1]);
            pf[rt][n][2 * j + i] = two;
            if (n + 1 < NP) {
              p_step[j][2 * i] -= bf16_bits_to_float(two & 0xFFFFu);
              p_step[j][2 * i + 1] -= bf16_bits_to_float(two >> 16);
            }
          }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if constexpr (NT > 1) of_step[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) of_step[rt] = product(ones, pf[rt][n], of_step[rt]);
    }
#pragma unroll
    for (int d = 0; d < C; ++d) {
      u32x4 vf;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          if constexpr (C == 2) vf[2 * j + pair] = codes(c.v[j][0], d + 2 * pair, mask);
          else vf[2 * j + pair] = codes(c.v[j][pair * (C / 4) + d / 4], d % 4, mask);
        }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) o[rt][d] = product(vf, pf[rt][n], o[rt][d]);
      // (in 32 bits sums are not left to grow by B + 8 beyond what they come to)
      if constexpr (NT > 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][d] -= (B + 8.f) * of_step[rt][0];
      }
    }
  };

  if (chunk_first < chunk_end) {
    // Page ids two chunks ahead, tokens one: the next chunk's keys and values take the registers of this one's as soon as these have been
    // used.  The two ways to take a chunk are loops of their own: a branch between them would keep the sums in two places.
    f32x4 s[RT][2];
    Chunk<HD> c;
    int chunk = chunk_first;
    Ids ids = ids_of(chunk), next = ids_of(chunk + W);
    request_keys(ids, c);
    request_values(ids, c);
    const unsigned whole_lo = max(all_lo, lo), whole_hi = min(all_hi, hi);
    const auto take = [&](auto whole) {
      const Ids after = ids_of(chunk + 2 * W);
      score(c, s);
      request_keys(next, c);
      add(whole, chunk, ids, c, s);
      request_values(next, c);
      chunk += W;
      ids = next;
      next = after;
    };
    const auto all_see = [&] {      // (the chunk's end may be 2^31)
      const unsigned t = static_cast<unsigned>(chunk) * kChunk;
      return t >= whole_lo && t + kChunk <= whole_hi && ids.some[0] && ids.some[1];
    };
    while (chunk < chunk_end) {
      while (all_see()) take(std::true_type());
      if (chunk < chunk_end) take(std::false_type());
    }
  }

  // Up to four waves at a time leave their sums in LDS; a row's lanes add them up, the waves in order.
  constexpr int AT_ONCE = W < 4 ? W : 4;
  __shared__ float os[AT_ONCE][16][HD + 4], ms[W][16], ls[W][16];
  constexpr int LANES = W * kWave / 16, PER = HD / LANES > 0 ? HD / LANES : 1;      // lanes of a row, entries of a lane
  const int r = threadIdx.x / LANES, at = threadIdx.x % LANES * PER;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float all = rows_sum(l[rt]), more = NT > 1 ? rows_sum(of_mid[rt]) : fmaf(-(B + 8.f), of_step[rt][0], rows_sum(of_mid[rt]));
    if (rt > 0) __syncthreads();
    if (kq == 0) {
      ms[wave][n16] = limit[rt] == -FLT_MAX ? -FLT_MAX : -less_m[rt][0];
      ls[wave][n16] = all;
    }
    float top = -FLT_MAX, sum = 0.f, x[PER] = {};
#pragma unroll
    for (int turn = 0; turn < W / AT_ONCE; ++turn) {
      if (turn > 0) __syncthreads();
      if (wave / AT_ONCE == turn) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < C; ++d) os[wave % AT_ONCE][n16][(4 * kq + i) * C + d] = o[rt][d][i] + more;
      }
      __syncthreads();
      if (turn == 0) {
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, ms[w][r]);
      }
#pragma unroll
      for (int w = 0; w < AT_ONCE; ++w) {
        const float by = __builtin_amdgcn_exp2f(ms[AT_ONCE * turn + w][r] - top);
        sum = fmaf(ls[AT_ONCE * turn + w][r], by, sum);
        if (at < HD) {
#pragma unroll
          for (int e = 0; e < PER; ++e) x[e] = fmaf(os[w][r][at + e], by, x[e]);
        }
      }
    }
    const int f = first + 16 * rt + r;
    if (f >= span.rows || at >= HD) continue;
    const int of = quotient(f, sh.group), h = kvh * group + f - of * group;
    const size_t to = span.row0 + of;
    if (segs > 1) {
      float* left = scratch + ((to * sh.nh + h) * sh.max_segs + part) * (HD + 2);
#pragma unroll
      for (int e = 0; e < PER; ++e) left[at + e] = x[e];
      if (at == 0) {
        left[HD] = top;
        left[HD + 1] = sum;
      }
    } else {
      const float by = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] *= by;
      store_some(out + to * sh.out_stride + h * HD + at, x);
    }
  }
}

// Joins the segments of a row: a workgroup a (row, head).  Each thread weighs a segment; 256 / HD threads share an entry, a
// segment in so many of them each, eight loads at a time under way.  (One wave that went through a row's 64 segments one after the other
// took 50 us.)
constexpr int kMostSegments = 1600;
template <class T, int HD>
__global__ void __launch_bounds__(256) join4_kernel(const float* __restrict__ scratch, T* __restrict__ out, Rows rows, Shape sh) {
  constexpr int G = 256 / HD, AHEAD = 8;
  __shared__ float weight[kMostSegments], sums[G][HD], of_wave[2][4];
  const int head = blockIdx.x, group = sh.group.d, wave = threadIdx.x / kWave;
  const Span span = span_of(rows, sh, blockIdx.z);
  const int at = blockIdx.y;      // position in the span
  if (at * group >= span.rows) return;
  const int f = at * group + head - quotient(head, sh.group) * group, block_first = f & ~(sh.tile_rows - 1);      // (tile_rows: a power of two)
  const int segs = cut_of(span, sh, block_first, min(block_first + sh.tile_rows, span.rows) - 1).segs;
  if (segs == 1) return;
  const size_t row = span.row0 + at;
  const float* left = scratch + (row * sh.nh + head) * sh.max_segs * (HD + 2);
  const int e = threadIdx.x % HD, g = threadIdx.x / HD;
  const auto some_of = [&](int i, float (&next)[AHEAD]) {
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) next[n] = i + n * G < segs ? left[static_cast<size_t>(i + n * G) * (HD + 2) + e] : 0.f;
  };
  // the first ones are under way while the weights are made
  float next[AHEAD];
  some_of(g, next);
  const int own = min(static_cast<int>(threadIdx.x), segs - 1) * (HD + 2) + HD;
  const float own_m = left[own], own_l = left[own + 1];
  float top = own_m, sum = 0.f;
  for (int i = threadIdx.x + 256; i < segs; i += 256) top = fmaxf(top, left[i * (HD + 2) + HD]);
  top = wave_max(top);
  if (threadIdx.x % kWave == 0) of_wave[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(of_wave[0][0], of_wave[0][1]), fmaxf(of_wave[0][2], of_wave[0][3]));
  for (int i = threadIdx.x; i < segs; i += 256) {
    const bool mine = i == static_cast<int>(threadIdx.x);
    const float by = __builtin_amdgcn_exp2f((mine ? own_m : left[i * (HD + 2) + HD]) - top);
    weight[i] = by;
    sum = fmaf(mine ? own_l : left[i * (HD + 2) + HD + 1], by, sum);
  }
  sum = wave_sum(sum);
  if (threadIdx.x % kWave == 0) of_wave[1][wave] = sum;
  __syncthreads();
  float x = 0.f;
  for (int i = g; i < segs; i += AHEAD * G) {
    if (i > g) some_of(i, next);
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) x = i + n * G < segs ? fmaf(next[n], weight[i + n * G], x) : x;
  }
  sums[g][e] = x;
  __syncthreads();
  if (g == 0) {
#pragma unroll
    for (int n = 1; n < G; ++n) x += sums[n][e];
    sum = (of_wave[1][0] + of_wave[1][1]) + (of_wave[1][2] + of_wave[1][3]);
    store_f(out + row * sh.out_stride + head * HD + e, sum == 0.f ? 0.f : x / sum);
  }
}

// ---- host side
struct Plan {
  int rt, waves, segment, max_segs, tile_rows, tiles;
  long long floats;
};

constexpr long long kFill = 768;      // workgroups that fill the chip: three on each of 256 CUs
static_assert(2 * kFill + 2 <= kMostSegments);

// What a call with its contexts cut into `parts` takes, roughly: a round of 128 tokens (a chunk of each wave) is 0.8 us where the chip is
// nearly empty and 2.5 where it is full; joining is a launch, the parts that a row's workgroup goes through, the workgroups, and the bytes.
// One row, 8 kv heads of 128: 8,192 tokens take 10.9 us in 64 parts and 9.0 in 32; 2,048 tokens 7.3 us in 16 and 7.8 in 8.  (All rows count as
// having the longest context, and all sequences the longest run: calls of unlike ones are cut less than they could be.)
double expected_us(long long parts, long long groups, long long rounds, long long T, int nh, int hd) {
  const long long passes = (groups * parts + kFill - 1) / kFill;
  const double load = static_cast<double>(groups * parts) / (passes * kFill), walk = passes * ((rounds + parts - 1) / parts) * (0.8 + 1.7 * load);
  return parts == 1 ? walk : walk + 2.5 + 0.07 * parts + static_cast<double>(T) * nh * (0.0008 + parts * (hd + 2) * 8 / 3e6);
}

Plan plan(bool wide, int units, int T, int max_run, int nh, int nkv, int hd, int max_context, int window) {
  Plan p{};
  const int group = nh / nkv;
  max_run = std::min(max_run, T);
  const long long pairs = static_cast<long long>(max_run) * group;
  constexpr int LEAST = 4 * kChunk;      // tokens of a round: a chunk of each wave
  long long groups, seen, rounds;
  const auto tile = [&](int rt) {
    p.rt = rt;
    p.tile_rows = 16 * rt;
    p.tiles = static_cast<int>((pairs + p.tile_rows - 1) / p.tile_rows);
    groups = static_cast<long long>(units) * nkv * p.tiles;
    seen = window > 0 ? std::min<long long>(static_cast<long long>(window) + p.tile_rows, max_context) : max_context;
    rounds = (seen + LEAST - 1) / LEAST;
  };
  // Two tiles of rows to a wave share its operands; one tile leaves twice as many workgroups, and is the faster while there is work for less than
  // two rounds of a full chip (32 heads over 8 of 128, one tile and two: four runs of 16 behind 500 tokens 7.2 us and 9.5, 16 of 64 behind 300
  // 21.8 and 16.1; over 4 of 64: a prompt of 256 5.1 and 6.0, of 2,048 55 and 42).  Float rows, whose terms take the registers, always one (over 8 of
  // 128, three runs of 300 behind 4,000 tokens 212 us and 669; over 4 of 64, a prompt of 2,048 78 and 73), and so 256 entries.
  p.waves = 4;
  tile(pairs > 16 && hd <= 128 && !wide ? 2 : 1);
  if (p.rt == 2 && groups * rounds < 2 * kFill) tile(1);
  // How many parts contexts are cut into: what the model makes least, among 1 2 3 4 6 8 12 16 .. and what fills the chip once.
  const long long most = std::min(2 * kFill / groups, rounds);
  long long parts = 1;
  double least = expected_us(1, groups, rounds, T, nh, hd);
  const auto consider = [&](long long n) {
    const double us = n > 1 && n <= most ? expected_us(n, groups, rounds, T, nh, hd) : least;
    if (us < least) least = us, parts = n;
  };
  for (long long n = 2; n <= most; n += n & (n - 1) ? n / 3 : n / 2) consider(n);
  consider(kFill / groups);
  // Few workgroups and up to 1,024 tokens: eight waves instead of four, and no parts (32 heads over 4 of 64, one row: 529 tokens 6.0 us, with
  // four waves 6.7; 1,000 tokens 7.8 us, in eight parts 6.7 and a second launch for the host).
  if (p.rt == 1 && hd <= 128 && groups <= 256 && rounds > 2 && seen <= 1024) {
    parts = 1;
    p.waves = 8;
  }
  // Many workgroups of few rounds: two waves, whose beginning and end (half of a short walk) are half as many (32 heads over 8 of 128: 128 rows
  // of 300 tokens 11.9 us, with four waves 14.8; 256 of 1,000 60.6 and 55.0.  Over 4 of 64: eight prompts of 128 tokens 8.2 us and 10.2, one of
  // 1,024 20.0 and 16.7).
  if (parts == 1 && groups >= 1024 && (p.rt == 1 ? 3 : 2) * seen <= groups) p.waves = 2;
  // Of 256 entries a CU holds four waves: two workgroups where there are enough (16 heads over 2: 200 rows of 300 tokens 12.0 us, with four
  // waves 17.1; a prompt of 2,048 92 and 110).
  if (parts == 1 && groups > 256 && hd == 256) p.waves = 2;
  p.segment = parts == 1 ? LEAST : static_cast<int>(std::max<long long>(LEAST, ((seen + parts - 1) / parts + LEAST - 1) / LEAST * LEAST));
  p.max_segs = parts == 1 ? 1 : static_cast<int>((static_cast<long long>(max_context) + p.segment - 1) / p.segment);
  if (parts > 1 && seen < max_context) p.max_segs = static_cast<int>((seen - 1) / p.segment + 2);
  p.floats = p.max_segs == 1 ? 0 : static_cast<long long>(T) * nh * p.max_segs * (hd + 2);
  return p;
}

long long scratch_floats(int units, int T, int max_run, int nh, int nkv, int hd, int max_context, int window) {      // for rows of either type
  return std::max(plan(false, units, T, max_run, nh, nkv, hd, max_context, window).floats, plan(true, units, T, max_run, nh, nkv, hd, max_context, window).floats);
}

int launch(const char* what, const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, const int* tables, int table_stride, Rows rows,
           int units, int max_run, int nh, int nkv, int hd, int pages, int page, float scale, int window, int max_context, float* scratch, long long scratch_floats,
           hipStream_t stream) {
  KVCM_REQUIRE(kvcm_cache4_supported(nh, nkv, hd, page), "%s: heads %d, kv heads %d, head_dim %d, pages of %d tokens are not taken", what, nh, nkv, hd, page);
  KVCM_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: dtype %d", what, dtype);
  KVCM_REQUIRE(pages > 0 && static_cast<long long>(pages) * page < (1ll << 31), "%s: %d pages of %d tokens", what, pages, page);
  KVCM_REQUIRE(table_stride > 0 && rows.seqs > 0 && static_cast<long long>(table_stride) * page < (1ll << 31), "%s: %d tables of %d pages", what, rows.seqs, table_stride);
  KVCM_REQUIRE(nh < 65536 && q_stride >= nh * hd && out_stride >= nh * hd && window >= 0 && max_context >= 0, "%s: rows of %d and %d entries, window %d, contexts up to %d",
               what, q_stride, out_stride, window, max_context);
  KVCM_REQUIRE(rows.total > 0 && max_run > 0, "%s: %d rows, runs of up to %d", what, rows.total, max_run);
  KVCM_REQUIRE(q != nullptr && out != nullptr && cache != nullptr && tables != nullptr && rows.where != nullptr && rows.lens != nullptr, "%s: null operand", what);
  max_run = std::min(max_run, rows.total);
  const Plan p = plan(dtype == kF32, units, rows.total, max_run, nh, nkv, hd, max_context, window);
  KVCM_REQUIRE(p.floats == 0 || (scratch != nullptr && scratch_floats >= p.floats), "%s: scratch of %lld floats is needed", what, p.floats);
  Shape s{};
  s.q_stride = q_stride, s.out_stride = out_stride, s.table_stride = table_stride, s.nh = nh, s.pages = pages;
  s.max_segs = p.max_segs, s.tiles = p.tiles, s.tile_rows = p.tile_rows;
  s.nkv = divisor(nkv), s.group = divisor(nh / nkv), s.segs = divisor(p.max_segs), s.page_tiles = divisor(page / kTile4), s.segment = divisor(p.segment / kChunk);
  s.scale_log2 = scale * 1.4426950408889634f;
  s.window = window, s.max_context = static_cast<int>(std::min<long long>(static_cast<long long>(table_stride) * page, max_context));
  const long long x = static_cast<long long>(nkv) * p.max_segs * p.tiles;
  // (2^32 threads of a launch in x, at most 512 of a workgroup; quotients below 2^30)
  KVCM_REQUIRE(x < (1ll << 23) && static_cast<long long>(rows.total) * (nh / nkv) < (1ll << 30) && units < 65536, "%s: %lld workgroups for each of %d sequences", what, x, units);
  KVCM_REQUIRE(p.max_segs == 1 || max_run < 65536, "%s: runs of %d rows cut into segments", what, max_run);
  const dim3 grid(static_cast<unsigned>(x), units);
  KVCM_HEAD4(hd, {
    auto go = [&](auto t) {
      using T = decltype(t);
      const T* qt = static_cast<const T*>(q);
      T* ot = static_cast<T*>(out);
      const uint8_t* ct = static_cast<const uint8_t*>(cache);
      const auto walk = [&](auto rt, auto waves) {
        constexpr int RT = decltype(rt)::value, W = decltype(waves)::value, RUNS = kTerms<T>, SINGLE = std::max(RUNS, 2);
        const auto kernel = rows.runs ? attention4_kernel<T, HD, RT, W, RUNS> : attention4_kernel<T, HD, RT, W, SINGLE>;
        kernel<<<grid, W * kWave, 0, stream>>>(qt, ot, ct, tables, rows, s, scratch);
      };
      constexpr std::integral_constant<int, 1> one;
      constexpr std::integral_constant<int, 4> four;
      constexpr std::integral_constant<int, 2> two;
      constexpr std::integral_constant<int, HD == 256 || sizeof(T) == 4 ? 1 : 2> most;
      if (p.rt == 2 && p.waves == 2) walk(most, two);
      else if (p.rt == 2) walk(most, four);
      else if (p.waves == 2) walk(one, two);
      else if (p.waves == 4) walk(one, four);
      else walk(one, std::integral_constant<int, HD == 256 ? 4 : 8>());
      if (p.max_segs > 1) join4_kernel<T, HD><<<dim3(nh, max_run, units), 256, 0, stream>>>(scratch, ot, rows, s);
    };
    if (dtype == kBF16) go(bf16_t());
    else go(float());
  });
  return launch_status(what);
}

}  // namespace
}  // namespace kvcm

using namespace kvcm;

extern "C" {

long long kvcm_attention_decode4_scratch(int T, int nh, int nkv, int hd, int max_context, int window) {
  if (T <= 0 || nkv <= 0 || nh <= 0 || nh % nkv != 0) return 0;
  return scratch_floats(T, T, 1, nh, nkv, hd, max_context, window);
}

int kvcm_attention_decode4(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, const int* tables, int table_stride, int seqs,
                           const int* row_seq, const int* ctx_lens, int T, int nh, int nkv, int hd, int pages, int page, float scale, int window, int max_context,
                           float* scratch, long long scratch_floats, hipStream_t stream) {
  if (T == 0) return 0;
  return launch("attention_decode4", q, dtype, q_stride, out, out_stride, cache, tables, table_stride, Rows{row_seq, ctx_lens, seqs, T, false}, T, 1, nh, nkv, hd, pages,
                page, scale, window, max_context, scratch, scratch_floats, stream);
}

long long kvcm_attention_prefill4_scratch(int T, int nh, int nkv, int hd, int max_context, int max_run, int num_seqs, int window) {
  if (T <= 0 || nkv <= 0 || nh <= 0 || nh % nkv != 0 || max_run <= 0 || num_seqs <= 0) return 0;
  return scratch_floats(num_seqs, T, max_run, nh, nkv, hd, max_context, window);
}

int kvcm_attention_prefill4(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, const int* tables, int table_stride,
                            const int* run_start, const int* seq_start, int num_seqs, int max_run, int T, int nh, int nkv, int hd, int pages, int page, float scale,
                            int window, int max_context, float* scratch, long long scratch_floats, hipStream_t stream) {
  if (T == 0 || num_seqs == 0 || max_run == 0) return 0;
  return launch("attention_prefill4", q, dtype, q_stride, out, out_stride, cache, tables, table_stride, Rows{run_start, seq_start, num_seqs, T, true}, num_seqs, max_run,
                nh, nkv, hd, pages, page, scale, window, max_context, scratch, scratch_floats, stream);
}

}  // extern "C"
