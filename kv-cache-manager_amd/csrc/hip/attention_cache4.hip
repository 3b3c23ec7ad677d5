// Attention over the 4-bit cache (cache4.h): softmax(scale * q . k) v over a row's visible tokens, max(0, p + 1 - window) <= t <= p.
//
// A wave takes one row of one head and walks its tokens 64 at a time with a running maximum m and sum l: a lane scores a token
// of its own, q . (low + step c) = low * sum(q) + step * (q . c), and then adds up entries of its own over the 64 tokens.
#include <cfloat>

#include "cache4.h"
#include "kvcm_hip.h"

namespace kvcm {
namespace {

template <class T, int HD, bool RUNS>
__global__ void __launch_bounds__(kWave) attention4_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, int out_stride,
                                                           const uint8_t* __restrict__ cache, const int* __restrict__ tables, int table_stride, int seqs,
                                                           const int* __restrict__ where, const int* __restrict__ lens, int nh, int nkv, int pages, int page,
                                                           float scale, int window) {
  __shared__ float qs[HD], ps[kWave];
  __shared__ const uint8_t* tiles_at[kWave];
  const int lane = threadIdx.x, head = blockIdx.y, kvh = head / (nh / nkv);
  long long row;
  int seq, ctx;
  if constexpr (RUNS) {
    seq = blockIdx.z;
    row = where[seq] + static_cast<int>(blockIdx.x);
    if (row >= where[seq + 1]) return;
    ctx = lens[seq] + static_cast<int>(blockIdx.x) + 1;
  } else {
    row = blockIdx.x;
    seq = where[row];
    ctx = static_cast<unsigned>(seq) < static_cast<unsigned>(seqs) ? lens[row] : 0;
  }
  ctx = min(ctx, table_stride * page);
  float sum_q = 0.f;
  for (int d = lane; d < HD; d += kWave) {
    qs[d] = load_f(q + row * q_stride + head * HD + d);
    sum_q += qs[d];
  }
  sum_q = wave_sum(sum_q);
  float m = -FLT_MAX, l = 0.f, o[(HD + kWave - 1) / kWave] = {};
  const int first = window > 0 ? max(0, ctx - window) : 0;
  for (int t0 = first; t0 < ctx; t0 += kWave) {
    const int t = t0 + lane;
    float s = -FLT_MAX;
    const uint8_t* tile = nullptr;
    if (t < ctx) {
      const unsigned pg = tables[static_cast<size_t>(seq) * table_stride + t / page];
      if (pg < static_cast<unsigned>(pages)) {
        tile = cache + ((static_cast<size_t>(pg) * nkv + kvh) * (page / kTile4) + t % page / kTile4) * tile4_bytes(HD);
        const int i = t % kTile4;
        float dot = 0.f;
        for (int w = 0; w < HD / 8; ++w) {
          const uint32_t c = reinterpret_cast<const uint32_t*>(tile + i * (HD / 2))[w];
          for (int n = 0; n < 8; ++n) dot = fmaf(qs[8 * w + n], static_cast<float>(c >> (4 * n) & 15u), dot);
        }
        const uint32_t pair = reinterpret_cast<const uint32_t*>(tile + 8 * HD)[i];
        s = scale * fmaf(step4(pair), dot, low4(pair) * sum_q);
      }
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float p = tile != nullptr ? expf(s - m_new) : 0.f, alpha = expf(m - m_new);
    m = m_new;
    l = l * alpha + wave_sum(p);
    __syncthreads();
    ps[lane] = p;
    tiles_at[lane] = tile;
    __syncthreads();
    for (int j = 0; j < (HD + kWave - 1) / kWave; ++j) {
      const int d = lane + j * kWave;
      o[j] *= alpha;
      if (d >= HD) continue;
      for (int k = 0; k < kWave; ++k) {
        if (tiles_at[k] == nullptr) continue;
        const uint8_t* values = tiles_at[k] + value4_at(HD);
        const int i = (t0 + k) % kTile4;
        const uint32_t pair = reinterpret_cast<const uint32_t*>(values + 8 * HD)[i];
        int at = value4_byte<HD>(i, d / 4);
        if constexpr (HD == 32) at += d % 4 / 2 * 4;
        else at += d % 4 / 2;
        o[j] = fmaf(ps[k], fmaf(step4(pair), static_cast<float>(values[at] >> (4 * (d % 2)) & 15), low4(pair)), o[j]);
      }
    }
  }
  for (int j = 0; j < (HD + kWave - 1) / kWave; ++j)
    if (lane + j * kWave < HD) store_f(out + row * out_stride + head * HD + lane + j * kWave, l == 0.f ? 0.f : o[j] / l);
}

}  // namespace
}  // namespace kvcm

using namespace kvcm;

namespace {

int check(const char* what, const void* q, int dtype, int q_stride, const void* out, int out_stride, const void* cache, const int* tables, int table_stride, int seqs,
          const int* a, const int* b, int nh, int nkv, int hd, int pages, int page, int window) {
  KVCM_REQUIRE(kvcm_cache4_supported(nh, nkv, hd, page), "%s: heads %d, kv heads %d, head_dim %d, pages of %d tokens are not taken", what, nh, nkv, hd, page);
  KVCM_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: dtype %d", what, dtype);
  KVCM_REQUIRE(pages > 0 && static_cast<long long>(pages) * page < (1ll << 31), "%s: %d pages of %d tokens", what, pages, page);
  KVCM_REQUIRE(table_stride > 0 && seqs > 0 && static_cast<long long>(table_stride) * page < (1ll << 31), "%s: %d tables of %d pages", what, seqs, table_stride);
  KVCM_REQUIRE(q_stride >= nh * hd && out_stride >= nh * hd && window >= 0 && nh < 65536 && seqs < 65536, "%s: rows of %d and %d entries, window %d", what, q_stride, out_stride, window);
  KVCM_REQUIRE(q != nullptr && out != nullptr && cache != nullptr && tables != nullptr && a != nullptr && b != nullptr, "%s: null operand", what);
  return 0;
}

}  // namespace

extern "C" {

long long kvcm_attention_decode4_scratch(int, int, int, int, int, int) { return 0; }

int kvcm_attention_decode4(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, const int* tables, int table_stride, int seqs,
                           const int* row_seq, const int* ctx_lens, int T, int nh, int nkv, int hd, int pages, int page, float scale, int window, int, float*,
                           long long, hipStream_t stream) {
  if (T == 0) return 0;
  if (check("attention_decode4", q, dtype, q_stride, out, out_stride, cache, tables, table_stride, seqs, row_seq, ctx_lens, nh, nkv, hd, pages, page, window)) return -1;
  KVCM_REQUIRE(T > 0, "attention_decode4: %d rows", T);
  KVCM_HEAD4(hd, {
    if (dtype == kBF16)
      attention4_kernel<bf16_t, HD, false><<<dim3(T, nh), kWave, 0, stream>>>(static_cast<const bf16_t*>(q), q_stride, static_cast<bf16_t*>(out), out_stride,
          static_cast<const uint8_t*>(cache), tables, table_stride, seqs, row_seq, ctx_lens, nh, nkv, pages, page, scale, window);
    else
      attention4_kernel<float, HD, false><<<dim3(T, nh), kWave, 0, stream>>>(static_cast<const float*>(q), q_stride, static_cast<float*>(out), out_stride,
          static_cast<const uint8_t*>(cache), tables, table_stride, seqs, row_seq, ctx_lens, nh, nkv, pages, page, scale, window);
  });
  return launch_status("attention_decode4");
}

long long kvcm_attention_prefill4_scratch(int, int, int, int, int, int, int, int) { return 0; }

int kvcm_attention_prefill4(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, const int* tables, int table_stride,
                            const int* run_start, const int* seq_start, int num_seqs, int max_run, int T, int nh, int nkv, int hd, int pages, int page, float scale,
                            int window, int, float*, long long, hipStream_t stream) {
  if (T == 0 || num_seqs == 0 || max_run == 0) return 0;
  if (check("attention_prefill4", q, dtype, q_stride, out, out_stride, cache, tables, table_stride, num_seqs, run_start, seq_start, nh, nkv, hd, pages, page, window)) return -1;
  KVCM_REQUIRE(T > 0 && max_run > 0, "attention_prefill4: %d rows, runs of up to %d", T, max_run);
  KVCM_HEAD4(hd, {
    if (dtype == kBF16)
      attention4_kernel<bf16_t, HD, true><<<dim3(max_run, nh, num_seqs), kWave, 0, stream>>>(static_cast<const bf16_t*>(q), q_stride, static_cast<bf16_t*>(out),
          out_stride, static_cast<const uint8_t*>(cache), tables, table_stride, num_seqs, run_start, seq_start, nh, nkv, pages, page, scale, window);
    else
      attention4_kernel<float, HD, true><<<dim3(max_run, nh, num_seqs), kWave, 0, stream>>>(static_cast<const float*>(q), q_stride, static_cast<float*>(out),
          out_stride, static_cast<const uint8_t*>(cache), tables, table_stride, num_seqs, run_start, seq_start, nh, nkv, pages, page, scale, window);
  });
  return launch_status("attention_prefill4");
}

}  // extern "C"
