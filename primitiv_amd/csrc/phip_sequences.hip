// Lengths of the sequences of a minibatch, made once per batch and read by every layer's rotary and attention calls.
#include <algorithm>
#include <new>
#include <vector>

#include "phip_sequences.h"

namespace phip {
namespace {

// The lists travel as kernel arguments: enqueued like any other work, with no wait of the host for the stream (a
// program that generates text makes a new list for every token).
constexpr uint32_t kPerLaunch = 64;
struct EntryChunk {
  SequenceEntry e[kPerLaunch];
};
struct PlaceChunk {
  SequencePlace p[kPerLaunch];
};

__global__ __launch_bounds__(kPerLaunch) void write_sequences_kernel(SequenceEntry *entries, SequencePlace *places,
                                                                     EntryChunk e, PlaceChunk p, uint32_t n) {
  const uint32_t i = threadIdx.x;
  if (i >= n) return;
  entries[i] = e.e[i];
  places[i] = p.p[i];
}

int create(phip_ctx *ctx, const uint32_t *q_lens, const uint32_t *k_lens, uint32_t n, bool packed,
           phip_sequences **out) {
  PHIP_ENTER(ctx);
  PHIP_REQUIRE(out != nullptr, "null output pointer");
  *out = nullptr;
  PHIP_REQUIRE(q_lens != nullptr, "null lengths");
  PHIP_REQUIRE(n >= 1 && n <= (1u << 24), "a list of 1 to 2^24 sequences is needed, got %u", n);
  if (k_lens == nullptr) k_lens = q_lens;
  std::vector<SequenceEntry> entries(n);
  std::vector<SequencePlace> places(n);
  uint64_t q_at = 0, k_at = 0;
  uint32_t max_q = 0, max_k = 0;
  for (uint32_t i = 0; i < n; ++i) {
    PHIP_REQUIRE(q_lens[i] <= 0x7fffffffu && k_lens[i] <= 0x7fffffffu, "sequence %u: a length above 2^31 - 1", i);
    entries[i] = {packed ? 0u : i, packed ? (uint32_t)q_at : 0u, q_lens[i], packed ? (uint32_t)k_at : 0u, k_lens[i], 0, 0, 0};
    places[i] = {entries[i].q_start, q_lens[i], (int32_t)k_lens[i] - (int32_t)q_lens[i], 0};
    q_at += q_lens[i];
    k_at += k_lens[i];
    if (packed) PHIP_REQUIRE(q_at <= 0x7fffffffu, "packed sequences of more than 2^31 - 1 queries");
    max_q = std::max(max_q, q_lens[i]);
    max_k = std::max(max_k, k_lens[i]);
  }
  std::stable_sort(entries.begin(), entries.end(), [](const SequenceEntry &a, const SequenceEntry &b) {
    return a.k_len != b.k_len ? a.k_len > b.k_len : a.q_len > b.q_len;
  });
  uint32_t q_cum = 0, k_cum = 0;  // read only where the totals fit
  for (SequenceEntry &e : entries) {
    e.q_cum = q_cum;
    e.k_cum = k_cum;
    q_cum += e.q_len;
    k_cum += e.k_len;
  }
  phip_sequences *s = new phip_sequences();
  s->ctx_id = ctx->id;
  s->n = n;
  s->packed = packed;
  s->max_q = max_q;
  s->max_k = max_k;
  s->q_total = packed ? (uint32_t)q_at : 0;
  s->k_sum = k_at;
  const int rc = phip_pool_alloc(ctx, (sizeof(SequenceEntry) + sizeof(SequencePlace)) * (size_t)n, &s->block, nullptr);
  if (rc != PHIP_OK) {
    delete s;
    return rc;
  }
  SequenceEntry *de = static_cast<SequenceEntry *>(s->block);
  SequencePlace *dp = reinterpret_cast<SequencePlace *>(de + n);
  for (uint32_t i = 0; i < n; i += kPerLaunch) {
    const uint32_t m = std::min(kPerLaunch, n - i);
    EntryChunk ec;
    PlaceChunk pc;
    std::copy(entries.begin() + i, entries.begin() + i + m, ec.e);
    std::copy(places.begin() + i, places.begin() + i + m, pc.p);
    hipLaunchKernelGGL(write_sequences_kernel, dim3(1), dim3(kPerLaunch), 0, ctx->stream, de + i, dp + i, ec, pc, m);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    phip_pool_free(ctx, s->block);
    delete s;
    return fail(PHIP_ERR_RUNTIME, "writing the list of sequences failed: %s", hipGetErrorString(e));
  }
  *out = s;
  return PHIP_OK;
}

}  // namespace

int sequence_view(phip_ctx *ctx, const phip_sequences *seqs, uint32_t tq, uint32_t tk, uint32_t bs, bool keys,
                  SequenceView *out) {
  if (seqs == nullptr) {
    *out = {nullptr, nullptr, bs, tq, tk, 0, 0, 0};
    return PHIP_OK;
  }
  PHIP_REQUIRE(seqs->ctx_id == ctx->id, "the list of sequences belongs to another context");
  if (seqs->packed) {
    PHIP_REQUIRE(bs == 1, "packed sequences lie in one sample, the tensors have %u", bs);
    PHIP_REQUIRE(seqs->q_total <= tq, "packed sequences of %u queries in %u tokens", seqs->q_total, tq);
    // operators that read no keys take any number of them: the lengths are positions there
    PHIP_REQUIRE(!keys || seqs->k_sum <= tk, "packed sequences of %llu keys in %u tokens", (unsigned long long)seqs->k_sum, tk);
  } else {
    PHIP_REQUIRE(seqs->n == bs, "%u sequences for %u samples", seqs->n, bs);
    PHIP_REQUIRE(seqs->max_q <= tq, "a sequence of %u queries in samples of %u tokens", seqs->max_q, tq);
    PHIP_REQUIRE(!keys || seqs->max_k <= tk, "a sequence of %u keys in samples of %u tokens", seqs->max_k, tk);
  }
  const SequenceEntry *e = static_cast<const SequenceEntry *>(seqs->block);
  *out = {e, reinterpret_cast<const SequencePlace *>(e + seqs->n), seqs->n, tq, tk, seqs->packed ? 1u : 0u,
          seqs->q_total, keys && seqs->packed ? (uint32_t)seqs->k_sum : 0};
  return PHIP_OK;
}

}  // namespace phip

extern "C" {

int phip_sequences_create(phip_ctx *ctx, const uint32_t *q_lens, const uint32_t *k_lens, uint32_t n, int packed,
                          phip_sequences **out) {
  try {
    return phip::create(ctx, q_lens, k_lens, n, packed != 0, out);
  } catch (const std::exception &) {
    return phip::fail(PHIP_ERR_OUT_OF_MEMORY, "out of host memory for a list of %u sequences", n);
  }
}

int phip_sequences_destroy(phip_sequences *seqs) {
  if (seqs == nullptr) return PHIP_OK;
  const int rc = phip_pool_free_by_id(seqs->ctx_id, seqs->block);
  delete seqs;
  return rc;
}

}  // extern "C"
