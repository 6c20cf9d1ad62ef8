// Launches of the token embedding and its gradient (embedding_kernel.hpp).
#include "embedding_kernel.hpp"
#include "layer_common.hpp"

namespace linrec {
namespace {

int check_embedding(const linrec_embedding_t* p) {
  if (!p || p->tokens < 0 || p->vocab < 0 || p->channels < 0 || (p->token_bytes != 4 && p->token_bytes != 8)) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->tokens > 2147483647LL - 8192 || p->vocab > 2147483647LL - 8192 || p->channels > 2147483647LL - 8192) return LINREC_E_TOO_LARGE;
  if (p->tokens > 0 && p->channels > 0 && !p->token) return LINREC_E_INVALID;
  return LINREC_OK;
}

// Channels of a lane: 16 bytes' worth, fewer where a row has no 64 such slots.
int slot_width(int dtype, int64_t channels) {
  int vec = dtype == LINREC_DTYPE_F32 ? 4 : 8;
  while (vec > 1 && channels < 64 * vec) vec >>= 1;
  return vec;
}
template <typename F>
int with_slot(int dtype, int64_t channels, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    switch (slot_width(dtype, channels)) {
      case 1: return f(t, std::integral_constant<int, 1>{});
      case 2: return f(t, std::integral_constant<int, 2>{});
      case 4: return f(t, std::integral_constant<int, 4>{});
    }
    if constexpr (sizeof(T) == 2) return f(t, std::integral_constant<int, 8>{});
    return int(LINREC_E_UNSUPPORTED);
  });
}

struct Scratch {
  size_t sorted[2], counts, runs, runs2, bytes;
  int64_t blocks, n_runs, n_runs2;
};
Scratch scratch_layout(int64_t tokens, int64_t channels) {
  Scratch s{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~size_t(255);
    return here;
  };
  const bool small = tokens <= SORT_SMALL;
  for (size_t& a : s.sorted) a = take(size_t(tokens) * 8);
  s.blocks = cdiv(tokens, SORT_BLOCK);
  s.counts = take(small ? 0 : size_t(s.blocks) * DIGITS * 4);
  s.n_runs = tokens / RUN;
  // (a launch more, 2 us for 32768 tokens of 32000, which have no such runs; without it 65536 tokens of 256 take 64 us instead of 43)
  s.n_runs2 = tokens < 16384 ? 0 : tokens / RUN2;
  s.runs = take(size_t(s.n_runs) * size_t(channels) * 4);
  s.runs2 = take(size_t(s.n_runs2) * size_t(channels) * 4);
  s.bytes = at;
  return s;
}

int bit_length(int64_t v) {
  int bits = 0;
  while (v >> bits) ++bits;
  return bits;
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

size_t linrec_embedding_scratch_bytes(int64_t tokens, int64_t, int64_t channels) {
  return tokens > 0 && channels > 0 ? scratch_layout(tokens, channels).bytes : 0;
}

int linrec_embedding_fwd(const linrec_embedding_t* p) {
  if (const int rc = check_embedding(p)) return rc;
  if (p->tokens == 0 || p->channels == 0) return LINREC_OK;
  if (!p->y || (p->vocab > 0 && !p->weight)) return LINREC_E_INVALID;
  return with_slot(p->dtype, p->channels, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    const int64_t column_waves = cdiv(p->channels, 64 * VEC);
    if (p->tokens * column_waves >= 16384)
      return launch_kernel(embedding_fwd_kernel<T, VEC, 4>, cdiv(cdiv(p->tokens, 4) * column_waves, 4), 1, 256, p->stream, *p, column_waves);
    return launch_kernel(embedding_fwd_kernel<T, VEC, 1>, cdiv(p->tokens * column_waves, 4), 1, 256, p->stream, *p, column_waves);
  });
}

int linrec_embedding_bwd(const linrec_embedding_t* p) {
  if (const int rc = check_embedding(p)) return rc;
  if (p->vocab == 0 || p->channels == 0) return LINREC_OK;
  if (!p->d_weight || (p->tokens > 0 && !p->d_y)) return LINREC_E_INVALID;
  const Scratch s = scratch_layout(p->tokens, p->channels);
  char* scratch = static_cast<char*>(p->scratch);
  if (p->tokens > 0 && (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15u) || p->scratch_bytes < s.bytes)) return LINREC_E_WORKSPACE;
  auto lists = [&](int i) {
    int* key = reinterpret_cast<int*>(scratch + s.sorted[i]);
    return Sorted{key, key + p->tokens};
  };
  // the gradient is cleared in equal shares by the sort's launches
  const int64_t bytes = p->vocab * p->channels * (p->dtype == LINREC_DTYPE_F32 ? 4 : 2), slots = bytes / 16;
  const int passes = int(cdiv(bit_length(p->vocab), DIGIT_BITS));  // (the key of what takes no part is `vocab`)
  const int shares = p->tokens <= SORT_SMALL ? 1 : 2 * passes;
  int share = 0;
  auto next_share = [&](int64_t* blocks) {
    Clear c{slots * share / shares, slots * (share + 1) / shares, 0};
    if (++share == shares) c.tail = int(bytes % 16 / 2);
    const int64_t n = cdiv(c.end - c.first, 4096);
    *blocks = n < 1 ? 1 : n > 256 ? 256 : n;
    return c;
  };
  Sorted sorted = lists(0);
  int64_t clearing;
  if (p->tokens <= SORT_SMALL) {
    const int64_t blocks = cdiv(p->tokens, SMALL_TAKE);
    const Clear c = next_share(&clearing);
    if (const int rc = launch_kernel(sort_small_kernel, blocks + clearing, 1, 1024, p->stream, *p, sorted, int(blocks), c)) return rc;
  } else {
    int* counts = reinterpret_cast<int*>(scratch + s.counts);
    const int* keys = nullptr;
    const int* positions = nullptr;
    for (int i = 0; i < passes; ++i) {
      sorted = lists(i & 1);
      Clear c = next_share(&clearing);
      if (const int rc = launch_kernel(digit_counts_kernel, s.blocks + clearing, 1, SORT_LANES, p->stream, *p, keys, i * DIGIT_BITS, counts, int(s.blocks), c))
        return rc;
      c = next_share(&clearing);
      if (const int rc = launch_kernel(digit_places_kernel, s.blocks + clearing, 1, SORT_LANES, p->stream, *p, keys, positions, i * DIGIT_BITS, counts,
                                       int(s.blocks), sorted, c))
        return rc;
      keys = sorted.key;
      positions = sorted.pos;
    }
  }
  if (p->tokens == 0) return LINREC_OK;
  return with_slot(p->dtype, p->channels, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int VEC = decltype(vec)::value;
    const int64_t column_waves = cdiv(p->channels, 64 * VEC);
    float* runs = reinterpret_cast<float*>(scratch + s.runs);
    float* runs2 = s.n_runs2 ? reinterpret_cast<float*>(scratch + s.runs2) : nullptr;
    if (const int rc = launch_kernel(run_sums_kernel<T, VEC, false>, cdiv(s.n_runs * column_waves, 4), 1, 256, p->stream, *p, sorted, nullptr, runs,
                                     s.n_runs, column_waves))
      return rc;
    if (const int rc = launch_kernel(run_sums_kernel<T, VEC, true>, cdiv(s.n_runs2 * column_waves, 4), 1, 256, p->stream, *p, sorted, runs, runs2,
                                     s.n_runs2, column_waves))
      return rc;
    return launch_kernel(list_sums_kernel<T, VEC>, cdiv(cdiv(p->tokens, OWN) * column_waves, 4), 1, 256, p->stream, *p, sorted, runs, runs2, column_waves);
  });
}

}  // extern "C"
