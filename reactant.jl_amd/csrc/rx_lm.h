// Operators of language models: what `stablehlo.custom_call` of an `rx.` target means, the checks of its operands and
// settings, and the launches that compute it.  The device code is kernels/rx_lm_kernels.h.
//
//   rx.embedding(table [V, D], ids [..]) {scale} -> [.., D]
//       out[t] = scale * table[ids[t]]; zeros where ids[t] is outside [0, V).
//   rx.embedding_grad(dy [.., D], ids [..]) {scale} -> [V, D]
//       the gradient of the table: scale * the sum of the rows of dy whose token is that row, summed in f32 in the order of the
//       tokens (the same bits every run); zeros for rows without tokens.
//   rx.kv_append(q [T, Hq, D], k [T, Hk, D], v [T, Hk, Dv], cos [L, R / 2], sin [L, R / 2], position [T], sequence [T],
//                pages [B, M], k_cache, v_cache) {rotation = "halves" | "pairs" | "none", layout = "slots" | "heads"}
//       -> (q', k_cache', v_cache')
//       Token t is at position p = position[t] of sequence b = sequence[t].  The first R dimensions of the heads of q and k are
//       rotated by the angles whose cosines and sines row p of the tables holds, as pairs (i, i + R / 2) ("halves") or
//       (2 i, 2 i + 1) ("pairs"); k and v go to slot p mod S of page pages[b, p div S], S being the slots of a page.  A
//       token whose p is outside [0, min(L, M S)) or whose b is outside [0, B) is padding: nothing is written for it and its
//       row of q' is zero.  A token whose page is outside the cache is not written.  No two tokens may name one slot.
//   rx.paged_attention(q [B, Hq, D], k_cache, v_cache, pages [B, M], lengths [B]) {scale, window, layout} -> out [B, Hq, Dv]
//                (or (out, lse [B, Hq] f32))
//       softmax(scale q k') v of one token per sequence over the positions [max(0, n - window), n) of its sequence (window = 0:
//       all), n = lengths[b] clamped to [0, M S].  Query head h reads head h div (Hq / Hk).  Positions on pages outside the cache
//       are left out.  Nothing left: out = 0, lse = -inf.  What lies in slots beyond a sequence is not looked at.  Scores of
//       positions in use that hold NaN or +inf give NaN; so do scores that are all -inf, with an lse of -inf.
//   rx.token_logprobs(logits [.., V], targets [..]) {top} -> (logprob, lse, entropy [, values [.., top], ids [.., top]])
//       log softmax at the target (0 where it is outside [0, V)), log of the sum of exponentials, entropy, and the `top`
//       largest log probabilities with their indices, largest first, equal ones by index.  -inf logits have probability 0; a row of
//       nothing else has lse = logprob = -inf and entropy 0, and its values are -inf.  A row with +inf or NaN has no probabilities:
//       its numbers are NaN, and its alternatives those of its logits, NaN before +inf.
//   rx.token_logprobs_grad(logits, targets, lse, entropy, d_logprob, d_entropy) -> d_logits
//
// Caches are [pages, S, Hk, D] (layout "slots") or [pages, Hk, S, D] ("heads").  Floats are f32, bf16 or f16, one type per operator
// except where noted; integers are i32 or i64.  Sums, statistics and products are carried in f32.
#pragma once
#include "rx_ir.h"

namespace rx {

struct OperatorSpec {
  std::string name;
  std::map<std::string, std::string> attrs;   // settings as written
  std::vector<TType> in, out;
};

struct OperatorArg {
  enum Kind { Operand, Result, Scratch, Counters } kind;
  int index;
};

struct OperatorKernel {
  std::string text;        // kernel text; "@K@" stands for the symbol's prefix
  std::string suffix;      // of the symbol
  std::string kind;
  unsigned grid[3] = {1, 1, 1};
  unsigned block = 256;
  std::vector<OperatorArg> args;   // what it writes last
  int n_outputs = 1;
  double bytes = 0, flops = 0;
};

struct OperatorPlan {
  std::vector<int64_t> scratch;    // bytes
  int64_t counters = 0;            // 32-bit words that live with the executable, zero before and after every launch
  std::vector<int> updates;        // per result: the operand that it is an updated copy of, or -1 (none: empty)
  std::vector<OperatorKernel> kernels;
};

bool is_operator_name(const std::string& name);
// Throws rx::Error where the operands, results or settings are not the operator's.
void check_operator(const OperatorSpec& spec);
// `lean`: with temporaries of up to 1 MiB for partial results (fewer workgroups share long sequences or rows).
OperatorPlan plan_operator(const OperatorSpec& spec, bool lean = false);
// Arithmetic of one call; *transcendentals: exponentials and logarithms, counted apart.
double operator_flops(const OperatorSpec& spec, double* transcendentals);

}  // namespace rx
