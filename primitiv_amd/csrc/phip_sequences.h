// The sequences of a minibatch: which tokens of a [.., heads, tokens] x batch tensor belong to which sequence.
#ifndef PHIP_SEQUENCES_H_
#define PHIP_SEQUENCES_H_

#include "phip_internal.h"

namespace phip {

// One sequence, as the attention kernels read it.  The entries are sorted by falling length (keys, then queries), so
// that the tiles of the longest sequences are launched first; q_cum and k_cum count the tokens of the entries before
// this one in that order (modulo 2^32; read only where the totals fit).
struct SequenceEntry {
  uint32_t sample;            // padded: which sample; packed: 0
  uint32_t q_start, q_len;    // first token (packed only, else 0) and number of tokens
  uint32_t k_start, k_len;    // (k_start: modulo 2^32, as k_cum)
  uint32_t q_cum, k_cum;
  uint32_t unused;
};

// The same in the order of the tokens, for operators that walk over them.
struct SequencePlace {
  uint32_t q_start, q_len;
  int32_t shift;              // k_len - q_len: the position of the sequence's first query
  uint32_t unused;
};

// What a kernel gets.  entries == nullptr: n samples of tq queries and tk keys each.
struct SequenceView {
  const SequenceEntry *entries;
  const SequencePlace *places;
  uint32_t n, tq, tk;
  uint32_t packed;
  uint32_t q_total, k_total;  // packed: tokens that belong to a sequence; those behind them belong to none

  __device__ inline SequenceEntry at(uint32_t i) const {
    if (entries != nullptr) return entries[i];
    return {i, 0, tq, 0, tk, 0, 0, 0};
  }
};

}  // namespace phip

struct phip_sequences {
  uint64_t ctx_id = 0;
  void *block = nullptr;  // n SequenceEntry, then n SequencePlace, on the device (context's pool)
  uint32_t n = 0;
  bool packed = false;
  uint32_t max_q = 0, max_k = 0;
  uint32_t q_total = 0;  // packed
  uint64_t k_sum = 0;    // keys of all sequences
};

namespace phip {

// The view of `seqs` (null: bs whole samples) on tensors of tq tokens (and tk keys, unless `keys` is false) and bs
// samples; checks that they fit.
int sequence_view(phip_ctx *ctx, const phip_sequences *seqs, uint32_t tq, uint32_t tk, uint32_t bs, bool keys,
                  SequenceView *out);

}  // namespace phip

#endif  // PHIP_SEQUENCES_H_
