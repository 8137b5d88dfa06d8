// Operators of language models: what `stablehlo.custom_call` of an `rx.` target means, the checks of its operands and
// settings, and the launches that compute it.  The device code is kernels/rx_lm_kernels.h, rx_lm_norm_kernels.h and rx_lm_cache_kernels.h.
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
//   rx.rms_norm(x [.., D] [, residual [.., D]], weight [D]) {eps} -> ([h,] y) or ([h,] y in 8 bits, scale [..])
//       h = x + residual (x itself without one), y = h weight / sqrt(mean(h^2) + eps), of h before it is rounded.  Squares are summed in f32.
//       1 <= D <= 32768.  (Without residual and 8 bits a reduction says the same, which becomes one launch of the generated code, a faster one.)
//   rx.rms_norm_grad(h [.., D], weight [D], dy [.., D] [, dh [.., D]]) {eps} -> (dx [.., D], dweight [D] in the type of h, or f32)
//       gradients by h (which is that by x and by residual) and by weight, for dy and dh arriving at y and h.
//   rx.kv_write(q [T, Hq, D], k [T, Hk, D], v [T, Hk, Dv], cos [L, R / 2], sin [L, R / 2], angle [A, T], position [T], sequence [T], pages [B, M],
//               k_cache, v_cache [, k_scale, v_scale]) {rotation, layout, sections} -> (q', k_cache', v_cache' [, k_scale', v_scale'])
//       rx.kv_append whose angles are told apart from the positions: token t goes to position[t] of sequence[t], and pair i of the rotated
//       dimensions is turned by row angle[a, t] of the tables, a the section that i lies in.  `sections` names the pairs of each of the A <= 4
//       axes ("16,24,24": time, height, width), in order; all R / 2 follow the one axis without it.  Caches of the type of k, or of 8 bits
//       with scales.  A token whose position is outside [0, M S), whose sequence is outside [0, B) or of whose rows one is outside [0, L)
//       (where it is turned) is padding: as for rx.kv_append.  No two tokens may name one slot.
//   rx.kv_move(lengths [B], path [B, A], pages [B, M], k_cache, v_cache [, k_scale, v_scale]) {layout} -> (k_cache', v_cache' [, k_scale', v_scale'])
//       Position lengths[b] + i of sequence b takes what position lengths[b] + path[b, i] held before the call: an accepted branch
//       moves together.  Not moved: where path[b, i] is negative, or either position is outside [0, M S) or on a page outside the cache.  A <= 64;
//       no two sequences may name one slot.
//   rx.tree_attention(q [B, N, Hq, D], k_cache, v_cache, pages [B, M], lengths [B] [, mask [N, N] or [B, N, N] i1] [, k_scale, v_scale])
//               {scale, window, layout} -> out [B, N, Hq, Dv] (or (out, lse [B, N, Hq] f32))
//       softmax(scale q k') v of N <= 1024 drafted tokens per sequence, which lie at positions lengths[b] .. lengths[b] + N - 1 of the cache.  Token i
//       sees the positions before lengths[b], and drafted token j where mask[.., i, j]; without a mask itself and those before it (N = 1: the
//       next token).  With a window (0: none, else at least N) a token sees that many positions: the drafted ones that it
//       sees, and the last of those before.  lengths[b] < 0: the sequence takes no part, and sees nothing.  Positions beyond M S and on pages outside
//       the cache are left out.  Nothing left: out = 0, lse = -inf.  What lies where a token does not see makes no difference to it.  An infinity or
//       NaN among the values that it sees gives it NaN or an infinity; scores as for rx.paged_attention.  Caches of q's type, or of 8 bits
//       with scales.
//
// Numbers of 8 bits (f8E4M3FN, or i8 from -127 to 127) stand for their product with a scale in f32, one for each row of a norm, or for each head's key
// and value of a position: scale = max(largest magnitude, 2^-100) / 448 (i8: 127), number = value / scale to nearest, ties to even.
// A row that holds an infinity or NaN has zeros and a scale of NaN.  Scales of caches are [pages, Hk, S] in either layout.  (An infinite scale of a key, which
// nothing here writes, makes its score an infinity or NaN.)
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
  std::string header = "rx_lm_kernels.h";   // of the device functions
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
