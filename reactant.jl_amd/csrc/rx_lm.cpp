// Checks and launches of the language-model operators (rx_lm.h).
#include "rx_lm.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <sstream>

namespace rx {
namespace {

struct OpName { const char* name; int in, out_min, out_max; };
const OpName kOperators[] = {
    {"rx.embedding", 2, 1, 1},       {"rx.embedding_grad", 2, 1, 1},  {"rx.kv_append", 10, 3, 3},
    {"rx.paged_attention", 5, 1, 2}, {"rx.token_logprobs", 2, 3, 5}, {"rx.token_logprobs_grad", 6, 1, 1},
};

constexpr int kMaxHeadDim = 256;
constexpr int64_t kMaxTop = 64;
constexpr int64_t kMaxGrid = (int64_t)1 << 22;   // workgroups; kernels with more items than that go on with the next ones
constexpr int64_t kLeanBytes = (int64_t)1 << 20;  // of partial results in a lean plan: a quarter of what calls without allocations have for all temporaries
constexpr int64_t kMaxRow = (int64_t)1 << 30;   // elements of a row or rows of a table: 32-bit indices inside a row

struct Checker {
  const OperatorSpec& s;
  [[noreturn]] void fail(const std::string& m) const { throw Error(s.name + ": " + m); }
  void require(bool ok, const std::string& m) const { if (!ok) fail(m); }
  void rank(const TType& t, int r, const char* what) const {
    require(t.rank() == r, std::string(what) + " must have " + std::to_string(r) + " dimensions, got " + t.str());
  }
  void floats(const TType& t, const char* what) const {
    require(t.dt == DT::F32 || t.dt == DT::BF16 || t.dt == DT::F16, std::string(what) + " must be f32, bf16 or f16, got " + t.str());
  }
  void f32(const TType& t, const char* what) const { require(t.dt == DT::F32, std::string(what) + " must be f32, got " + t.str()); }
  void ints(const TType& t, const char* what) const {
    require(t.dt == DT::I32 || t.dt == DT::I64, std::string(what) + " must be i32 or i64, got " + t.str());
  }
  void same(const TType& a, const TType& b, const char* what) const { require(a == b, std::string(what) + ": " + a.str() + " and " + b.str() + " differ"); }
  void dims(const TType& t, const std::vector<int64_t>& d, const char* what) const {
    TType w = t;
    w.dims = d;
    require(t.dims == d, std::string(what) + " must be " + w.str() + ", got " + t.str());
  }
  void settings(const std::set<std::string>& known) const {
    for (auto& kv : s.attrs) require(known.count(kv.first) != 0, "unknown setting '" + kv.first + "'");
  }
  double number(const char* key, double otherwise) const {
    auto it = s.attrs.find(key);
    if (it == s.attrs.end()) return otherwise;
    char* end = nullptr;
    const double v = std::strtod(it->second.c_str(), &end);
    require(end && *end == 0 && end != it->second.c_str() && std::isfinite(v), std::string("setting '") + key + "' must be a finite number, got '" + it->second + "'");
    return v;
  }
  // a factor that the kernels hold in f32, `times` another
  void scale(double times = 1.0) const {
    const double v = number("scale", 1.0);
    require(std::fabs(v * times) <= 3.4028234e38, "setting 'scale' must be a number that f32 holds" + std::string(times > 1 ? " times log2 e" : "") + ", got '" +
                                                     (s.attrs.count("scale") ? s.attrs.at("scale") : std::string()) + "'");
  }
  int64_t integer(const char* key, int64_t otherwise) const {
    const double v = number(key, (double)otherwise);
    require(v == std::floor(v) && std::fabs(v) < 1e15, std::string("setting '") + key + "' must be a whole number");
    return (int64_t)v;
  }
  std::string word(const char* key, const std::string& otherwise, const std::set<std::string>& known) const {
    auto it = s.attrs.find(key);
    const std::string v = it == s.attrs.end() ? otherwise : it->second;
    std::string all;
    for (auto& k : known) all += (all.empty() ? "'" : ", '") + k + "'";
    require(known.count(v) != 0, std::string("setting '") + key + "' must be one of " + all + ", got '" + v + "'");
    return v;
  }
};

struct Cache {   // [pages, slots of a page, heads, dim] or [pages, heads, slots, dim]
  int64_t pages, slots, heads, dim;
  bool by_slot;
  Cache(const TType& t, bool slots_first) : pages(t.dims[0]), slots(t.dims[slots_first ? 1 : 2]), heads(t.dims[slots_first ? 2 : 1]), dim(t.dims[3]), by_slot(slots_first) {}
};

std::vector<int64_t> without_last(const TType& t) { return std::vector<int64_t>(t.dims.begin(), t.dims.end() - 1); }
int64_t product(const std::vector<int64_t>& d) {
  int64_t n = 1;
  for (int64_t x : d) n *= x;
  return n;
}

const char* elem(DT t) { return t == DT::F32 ? "rx_lm_f32" : t == DT::BF16 ? "rx_lm_bf16" : "rx_lm_f16"; }
std::string num(int64_t v) { return std::to_string(v); }
std::string flt(double v) {
  char b[40];
  snprintf(b, sizeof b, "%.9g", v);
  std::string s = b;
  if (s.find_first_of(".en") == std::string::npos) s += ".0";
  return s + "f";
}

// `body` is the call of a device function on a0, a1, ..: the kernel's parameters, of which the last `outs` are written.
// `waves`: wavefronts per SIMD that the registers have to allow (0: the compiler's choice)
OperatorKernel kernel(const OperatorSpec& s, const std::string& suffix, unsigned block, const std::vector<std::pair<OperatorArg, std::string>>& args, int outs,
                      const std::string& body, int waves = 0) {
  OperatorKernel k;
  k.suffix = suffix;
  k.kind = "lm_" + suffix;
  k.block = block;
  k.n_outputs = outs;
  std::ostringstream o;
  o << "// " << s.name;
  for (auto& t : s.in) o << " " << t.str();
  o << "\nextern \"C\" __global__ __launch_bounds__(" << block << (waves ? ", " + num(waves) : std::string()) << ") void @K@_" << suffix << "(";
  for (size_t a = 0; a < args.size(); ++a) {
    const bool in = a + (size_t)outs < args.size();
    o << (a ? ", " : "") << (in ? "const " : "") << args[a].second << "* __restrict__ a" << a;
    k.args.push_back(args[a].first);
  }
  o << ") {\n  " << body << "\n}\n\n";
  k.text = o.str();
  return k;
}
OperatorArg operand(int i) { return {OperatorArg::Operand, i}; }
OperatorArg result(int i) { return {OperatorArg::Result, i}; }
OperatorArg scratch(int i) { return {OperatorArg::Scratch, i}; }
OperatorArg counters() { return {OperatorArg::Counters, 0}; }
std::string st(const TType& t) { return info(t.dt).stype; }

// ------------------------------------------------------------------ embedding
void check_embedding(const Checker& c) {
  const TType &table = c.s.in[0], &ids = c.s.in[1], &out = c.s.out[0];
  c.settings({"scale"});
  c.scale();
  c.rank(table, 2, "the table");
  c.floats(table, "the table");
  c.ints(ids, "ids");
  std::vector<int64_t> d = ids.dims;
  d.push_back(table.dims[1]);
  c.dims(out, d, "the result");
  c.require(out.dt == table.dt, "the result must have the table's type");
  c.require(table.dims[0] <= kMaxRow && table.dims[1] <= kMaxRow, "the table is too large");
  c.require(ids.numel() <= kMaxRow, "too many tokens");
}
OperatorPlan plan_embedding(const OperatorSpec& s) {
  const Checker c{s};
  const int64_t V = s.in[0].dims[0], D = s.in[0].dims[1], T = s.in[1].numel();
  OperatorPlan p;
  const int vec = (int)(16 / info(s.in[0].dt).size);
  const bool whole = D % vec == 0;
  const int64_t per = whole ? vec : 1, each = 2;   // vectors of a thread: 16384 rows of 4096 bf16 55 us with one, 32 with two, 34 with four
  OperatorKernel k = kernel(s, "embedding", 256, {{operand(0), st(s.in[0])}, {operand(1), st(s.in[1])}, {result(0), st(s.out[0])}}, 1,
                            std::string("rx_embedding<") + elem(s.in[0].dt) + ", " + num(V) + ", " + num(D) + ", " + num(T) + ", " + num(whole ? vec : 1) + ", " + num(each) +
                                ">(a0, a1, a2, " + flt(c.number("scale", 1.0)) + ");");
  k.grid[0] = (unsigned)std::min<int64_t>((T * (D / per) + 256 * each - 1) / (256 * each), kMaxGrid);
  k.bytes = (double)(2 * s.out[0].bytes() + s.in[1].bytes());
  p.kernels.push_back(k);
  return p;
}

void check_embedding_grad(const Checker& c) {
  const TType &dy = c.s.in[0], &ids = c.s.in[1], &out = c.s.out[0];
  c.settings({"scale"});
  c.scale();
  c.floats(dy, "dy");
  c.ints(ids, "ids");
  c.require(dy.rank() >= 1, "dy must have a dimension");
  c.rank(out, 2, "the result");
  c.floats(out, "the result");
  c.require(out.dt == dy.dt || out.dt == DT::F32, "the result must have the type of dy, or be f32");
  std::vector<int64_t> d = ids.dims;
  d.push_back(out.dims[1]);
  c.dims(dy, d, "dy");
  c.require(out.dims[0] <= kMaxRow && out.dims[1] <= kMaxRow, "the table is too large");
  c.require(ids.numel() <= kMaxRow, "too many tokens");
}
OperatorPlan plan_embedding_grad(const OperatorSpec& s, bool lean) {
  const Checker c{s};
  const int64_t V = s.out[0].dims[0], D = s.out[0].dims[1], T = s.in[1].numel();
  const std::string scale = flt(c.number("scale", 1.0)), types = std::string(elem(s.in[0].dt)) + ", " + elem(s.out[0].dt) + ", ";
  const int64_t wide = 16 / info(s.out[0].dt).size, vec = D % wide == 0 ? wide : 1, C = D / vec;   // a thread writes 16 bytes
  const int64_t rows_grid = std::min<int64_t>((V * C + 255) / 256, kMaxGrid);
  OperatorPlan p;
  if (rows_grid == 0) return p;
  // Up to 768 tokens in one launch without a sorted list (rows x dimensions of 5003 x 1024 f32, 32000 x 1024 bf16 and 512 x 768 f32:
  // with 512 tokens 9.3, 12.7 and 9.9 us against 12.0, 17.9 and 11.6 in two; with 768 11.0, 14.9 and 12.7 against 11.7, 18.2 and 11.4;
  // with 1024 13.1, 16.5 and 17.0 against 12.3, 19.0 and 11.4).
  if (T <= (V < 4096 ? 512 : 768)) {
    const std::string sizes = num(V) + ", " + num(D) + ", " + num(std::max<int64_t>(T, 1)) + ", " + num(vec);
    OperatorKernel k = T == 0 ? kernel(s, "embedding_grad", 256, {{result(0), st(s.out[0])}}, 1, "rx_lm_zero<" + num(V * D) + ">(a0);")
                              : kernel(s, "embedding_grad", 256, {{operand(0), st(s.in[0])}, {operand(1), st(s.in[1])}, {result(0), st(s.out[0])}}, 1,
                                       "rx_embedding_grad_few<" + types + sizes + ">(a0, a1, a2, " + scale + ");");
    const int64_t lines = C < 1024 ? 1024 / C : 1;
    k.grid[0] = (unsigned)(T == 0 ? rows_grid : std::min<int64_t>((V + lines - 1) / lines, kMaxGrid));
    k.bytes = (double)(s.in[0].bytes() + s.in[1].bytes() + s.out[0].bytes());
    p.kernels.push_back(k);
    return p;
  }
  // 256 workgroups sort, or as many as keep their rows' counters in LDS
  const int64_t rows = std::min<int64_t>(512, (V + 255) / 256);
  const int64_t parts = lean ? std::max<int64_t>(1, std::min<int64_t>(256, kLeanBytes / (8 * D))) : 256;
  const int64_t piece = std::max<int64_t>(64, (T + parts - 1) / parts), pieces = (T + piece - 1) / piece, tiles = (C + 255) / 256;
  p.scratch = {(V + 1) * 4, T * 4, T * 4, pieces * 2 * D * 4};
  OperatorKernel k = kernel(s, "embedding_sort", 1024, {{operand(1), st(s.in[1])}, {scratch(0), "int"}, {scratch(1), "int"}, {scratch(2), "int"}}, 3,
                            "rx_lm_sort<" + num(V) + ", " + num(T) + ", " + num(rows) + ">(a0, a1, a2, a3);");
  k.grid[0] = (unsigned)((V + rows - 1) / rows);
  p.kernels.push_back(k);
  // vectors of a row to a thread (16384 bf16 tokens, 65536 x 4096 f32: one 244 us, two 232, four 245)
  const int64_t each = std::min<int64_t>(2, tiles), wide_tiles = (C + 256 * each - 1) / (256 * each), lines = C < 256 ? 256 / C : 1;
  const std::string sizes = types + num(V) + ", " + num(D) + ", " + num(T) + ", " + num(vec) + ", " + num(piece);
  p.counters = pieces * wide_tiles;
  k = kernel(s, "embedding_grad", 256,
             {{operand(0), st(s.in[0])}, {scratch(0), "int"}, {scratch(1), "int"}, {scratch(2), "int"}, {result(0), st(s.out[0])}, {scratch(3), "float"}, {counters(), "int"}}, 3,
             "rx_embedding_grad_rows<" + sizes + ", " + num(each) + ">(a0, a1, a2, a3, a4, a5, a6, " + scale + ");");
  k.grid[0] = (unsigned)(std::min<int64_t>((V + lines - 1) / lines * wide_tiles, kMaxGrid) + pieces * wide_tiles);
  k.bytes = (double)(s.in[0].bytes() + s.in[1].bytes() + s.out[0].bytes());
  p.kernels.push_back(k);
  return p;
}

// ------------------------------------------------------------------ paged cache
void check_caches(const Checker& c, const TType& k, const TType& v, const TType& pages, bool by_slot) {
  c.rank(k, 4, "k_cache");
  c.rank(v, 4, "v_cache");
  c.floats(k, "k_cache");
  c.require(v.dt == k.dt, "the caches must have one type");
  const Cache kc(k, by_slot), vc(v, by_slot);
  c.require(kc.pages == vc.pages && kc.slots == vc.slots && kc.heads == vc.heads, "the caches must have the same pages, slots and heads: " + k.str() + " and " + v.str());
  c.require(kc.dim >= 1 && kc.dim <= kMaxHeadDim && vc.dim >= 1 && vc.dim <= kMaxHeadDim, "head dimensions from 1 to " + num(kMaxHeadDim) + " are supported");
  c.require(kc.slots >= 1 && kc.slots <= kMaxRow && kc.heads >= 1, "a cache's pages must have slots and heads");
  c.require(kc.pages <= kMaxRow, "the cache has too many pages");
  c.rank(pages, 2, "the page table");
  c.ints(pages, "the page table");
  c.require(pages.dims[1] * kc.slots <= kMaxRow && pages.dims[1] <= kMaxRow, "the page table's positions are too many");
}
void check_append(const Checker& c) {
  const auto& in = c.s.in;
  c.settings({"rotation", "layout"});
  const std::string rotation = c.word("rotation", "halves", {"halves", "pairs", "none"});
  const bool by_slot = c.word("layout", "slots", {"slots", "heads"}) == "slots";
  for (int i = 0; i < 3; ++i) {
    c.rank(in[i], 3, i == 0 ? "q" : i == 1 ? "k" : "v");
    c.floats(in[i], i == 0 ? "q" : i == 1 ? "k" : "v");
    c.require(in[i].dt == in[0].dt, "q, k and v must have one type");
  }
  check_caches(c, in[8], in[9], in[7], by_slot);
  c.require(in[8].dt == in[0].dt, "the caches must have the type of k");
  const Cache kc(in[8], by_slot), vc(in[9], by_slot);
  const int64_t T = in[0].dims[0];
  c.dims(in[0], {T, in[0].dims[1], kc.dim}, "q");
  c.dims(in[1], {T, kc.heads, kc.dim}, "k");
  c.dims(in[2], {T, kc.heads, vc.dim}, "v");
  c.f32(in[3], "cos");
  c.same(in[3], in[4], "cos and sin");
  c.rank(in[3], 2, "cos");
  c.require(in[3].dims[0] <= kMaxRow, "too many positions");
  c.require(rotation == "none" || 2 * in[3].dims[1] <= kc.dim, "the rotated dimensions exceed the head's: " + in[3].str() + " for heads of " + num(kc.dim));
  c.ints(in[5], "position");
  c.dims(in[5], {T}, "position");
  c.same(in[5], in[6], "position and sequence");
  c.require(in[7].dt == in[5].dt, "position, sequence and the page table must have one type");
  c.same(c.s.out[0], in[0], "q and its result");
  c.same(c.s.out[1], in[8], "k_cache and its result");
  c.same(c.s.out[2], in[9], "v_cache and its result");
  c.require(T <= kMaxRow && in[0].dims[1] <= (1 << 20) && kc.heads <= (1 << 20), "too many tokens or heads");
}
OperatorPlan plan_append(const OperatorSpec& s) {
  const Checker c{s};
  const auto& in = s.in;
  const bool by_slot = c.word("layout", "slots", {"slots", "heads"}) == "slots";
  const std::string rotation = c.word("rotation", "halves", {"halves", "pairs", "none"});
  const Cache kc(in[8], by_slot), vc(in[9], by_slot);
  const int64_t T = in[0].dims[0], R2 = rotation == "none" ? 0 : in[3].dims[1];
  OperatorPlan p;
  p.updates = {-1, 8, 9};
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < 8; ++i) args.push_back({operand(i), st(in[i])});
  for (int i = 0; i < 3; ++i) args.push_back({result(i), st(s.out[i])});
  std::ostringstream b;
  const int64_t ne = 16 / info(in[0].dt).size, HQ = in[0].dims[1];
  const bool pairs = rotation == "pairs", whole = kc.dim % ne == 0 && vc.dim % ne == 0 && 2 * R2 % ne == 0 && (pairs || R2 % ne == 0);
  // two heads of the same dimensions to a thread, their cosines and sines loaded once, where there are threads enough: 8191 tokens of
  // 40 heads of 128, half of it rotated, 42 -> 38 us, all of it 36.6 both; 512 tokens 4.1 -> 4.6, 48 tokens 2.8 -> 3.4
  const int64_t heads = T >= 2048 ? 2 : 1;
  b << (whole ? "rx_kv_append<" : "rx_kv_append_any<") << elem(in[0].dt) << ", " << HQ << ", " << kc.heads << ", " << kc.dim << ", " << vc.dim << ", " << kc.pages << ", " << kc.slots << ", "
    << in[7].dims[0] << ", " << in[7].dims[1] << ", " << in[3].dims[0] << ", " << R2 << ", " << (pairs ? "true" : "false") << ", " << (by_slot ? "true" : "false") << ", " << T
    << (whole ? ", " + num(heads) : std::string()) << ">(a0, a1, a2, a3, a4, a5, a6, a7, a8, a9, a10);";
  OperatorKernel k = kernel(s, "kv_append", 256, args, 3, b.str());
  const int64_t units = (pairs ? 2 * R2 : R2) / ne + (kc.dim - 2 * R2) / ne;
  const int64_t all = ((HQ + heads - 1) / heads + (kc.heads + heads - 1) / heads) * units + (kc.heads * vc.dim / ne + heads - 1) / heads;
  k.grid[0] = (unsigned)std::min<int64_t>(whole ? (T * all + 255) / 256 : T, kMaxGrid);
  k.bytes = 2.0 * (double)(in[0].bytes() + in[1].bytes() + in[2].bytes()) + 8.0 * (double)(T * R2) + (double)(in[5].bytes() * 3);
  p.kernels.push_back(k);
  return p;
}

// ------------------------------------------------------------------ attention
void check_attention(const Checker& c) {
  const auto& in = c.s.in;
  c.settings({"scale", "window", "layout"});
  const bool by_slot = c.word("layout", "slots", {"slots", "heads"}) == "slots";
  c.rank(in[0], 3, "q");
  c.floats(in[0], "q");
  check_caches(c, in[1], in[2], in[3], by_slot);
  c.require(in[1].dt == in[0].dt, "the caches must have the type of q");
  const Cache kc(in[1], by_slot), vc(in[2], by_slot);
  const int64_t B = in[0].dims[0], Hq = in[0].dims[1];
  c.require(in[0].dims[2] == kc.dim, "q and k_cache must have the same head dimension");
  c.require(Hq >= 1 && Hq % kc.heads == 0, "the query heads (" + num(Hq) + ") must be a multiple of the cache's (" + num(kc.heads) + ")");
  c.dims(in[3], {B, in[3].dims[1]}, "the page table");
  c.ints(in[4], "lengths");
  c.dims(in[4], {B}, "lengths");
  c.require(in[4].dt == in[3].dt, "lengths and the page table must have one type");
  c.dims(c.s.out[0], {B, Hq, vc.dim}, "the result");
  c.require(c.s.out[0].dt == in[0].dt, "the result must have the type of q");
  if (c.s.out.size() == 2) {
    c.f32(c.s.out[1], "lse");
    c.dims(c.s.out[1], {B, Hq}, "lse");
  }
  c.scale(1.4426950408889634);
  c.require(c.integer("window", 0) >= 0, "the window must not be negative");
  c.require(B <= 65535 && Hq <= 65535, "too many sequences or heads");
  c.require(B * Hq * std::max<int64_t>(vc.dim, 1) <= kMaxRow, "too many sequences and heads");
}
OperatorPlan plan_attention(const OperatorSpec& s, bool lean) {
  const Checker c{s};
  const auto& in = s.in;
  const bool by_slot = c.word("layout", "slots", {"slots", "heads"}) == "slots";
  const Cache kc(in[1], by_slot), vc(in[2], by_slot);
  const int64_t B = in[0].dims[0], Hq = in[0].dims[1], M = in[3].dims[1];
  const double scale = c.number("scale", 1.0 / std::sqrt((double)kc.dim));
  const int64_t window = std::min<int64_t>(c.integer("window", 0), kMaxRow);
  const bool lse = s.out.size() == 2;
  // A wavefront takes up to 32 query heads of a key head: 64 of one key head over 16 sequences of 61035 positions in bf16 take 293 us
  // in tiles of 16, 166 us in tiles of 32, 181 us in one of 64; of more than 128 dimensions tiles of 32 do not fit the registers.
  // Registers of a wavefront: a step's keys and values, the queries, the result, and room for the rest, of which 32-bit values need
  // less.  Up to 256 of them two wavefronts share a SIMD, and two workgroups a compute unit: 8 heads of 128 dimensions in f32, an
  // estimate of 216, 94 us with two and 102 with one; 32 heads in bf16, an estimate of 208, 145 and 118.
  const int64_t e = info(in[0].dt).size, ne = 16 / e, nk = (kc.dim + 4 * ne - 1) / (4 * ne), nv = (vc.dim + 16 * ne - 1) / (16 * ne);
  const int64_t G = Hq / kc.heads;
  auto registers = [&](int64_t n) { return 8 * nk + 32 * nv + n * (4 * nk + 4 * nv * ne + 24); };
  // One f32 query head per key head on the vector units: 12 heads of 80 dimensions, 7 sequences of up to 4001 positions, 20.6 -> 17.4
  // us; 16 sequences of 2288 positions, 8 heads of 128, 59 -> 55 us.  Two would gain 1 in 60, four lose as much.
  const bool vector = e == 4 && G == 1;
  const int64_t NT = G > 16 && registers(2) < 320 ? 2 : 1;
  const int64_t tiles = (G + 16 * NT - 1) / (16 * NT), GT = std::min(G, 16 * NT);
  const int waves = registers(NT) <= (e == 4 ? 230 : 196) ? 2 : 1;
  const int64_t longest = window ? std::min(M * kc.slots, window + 31) : M * kc.slots, units = std::max<int64_t>(1, (longest + 31) / 32);
  // A position's heads lie next to one another in a cache of slots: two heads to a workgroup read longer runs (16 sequences, 8 key
  // heads of 128 and 64 dimensions in bf16: 5.3 -> 5.7 and 4.5 -> 5.0 TB/s; four heads 5.6 and 5.0).  Its parts of long sequences are
  // twice as many, which costs more where a key head has many query heads, and where there may be few positions.
  const int64_t HW = by_slot && kc.heads % 2 == 0 && kc.heads >= 4 && kc.dim * e <= 256 && G <= 8 && B * units * kc.heads >= 4096 && !lean ? 2 : 1;
  // Rows of whole 256 bytes are read once and past the L2 (4.3 GB: 717 -> 630 us); of others it holds the lines that two reads share
  // (rows of 160 bytes, one head to a workgroup: 4.1 TB/s against 3.4), and better so where the neighbouring heads' workgroups are on
  // one die (4.6).  So it is with the tiles of one key head (64 query heads: 194 us past the L2, 171 through it, 166 on one die).
  const bool once = kc.dim * e % 256 == 0 && vc.dim * e % 256 == 0 && tiles == 1, dies = (by_slot && kc.dim * e % 128 != 0) || tiles > 1;
  const int64_t columns = kc.heads / HW * tiles;
  // Workgroups: all on the chip at once (half as many again: 64 sequences of 1 to 8192 positions 56 -> 60 us, one of 131072 630 -> 638),
  // two to a compute unit where the registers allow it; but one where each reads two heads' rows of 256 bytes, whose loads are enough
  // in flight (64 sequences of 1000 positions in bf16 55.7 -> 46.8 us, of 1 to 8192 56.1 -> 52.5; 64 dimensions of f32, 4 query heads a
  // key head, 56.4 -> 49.0; with rows of 128 bytes 59 -> 68, with one head to a workgroup 45.0 -> 48.5).  Shorter rows keep two: 64 uneven
  // sequences and 16 of 16384, 8 key heads in bf16, two and one: 128 bytes 29 and 36, 108 and 133 us; 160: 44 and 51, 137 and 159; 192: 48 and
  // 53, 155 and 167; 224: 57 and 60, 180 and 185; 256: 56 and 52, 180 and 175; f32 of 160 and 192 bytes 47 and 57, 141 and 186; 49 and 60, 155 and 192.
  const int64_t room = 256 * (HW == 2 && kc.dim * e == 256 ? 1 : waves);
  // every workgroup a stretch of at least four units of 32 positions (a sequence counts four more), all of them on the chip at once
  const int64_t part = 2 * HW * GT * (vc.dim * 4 + 8), most = lean ? std::min<int64_t>(room, kLeanBytes / part) : room;
  const int64_t stretches = std::max<int64_t>(1, std::min(most / columns, (B * (units + (B > 1 ? 4 : 0)) + 3) / 4)), grid = stretches * columns;
  OperatorPlan p;
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < 5; ++i) args.push_back({operand(i), st(in[i])});
  args.push_back({result(0), st(s.out[0])});
  if (lse) args.push_back({result(1), "float"});
  std::string shared = "(float*)0, (float*)0, (int*)0";
  if (stretches > 1) {
    p.scratch = {grid * 2 * HW * GT * vc.dim * 4, grid * 2 * HW * GT * 8};
    p.counters = B * columns;
    args.push_back({scratch(0), "float"});
    args.push_back({scratch(1), "float"});
    args.push_back({counters(), "int"});
    shared = lse ? "a7, a8, a9" : "a6, a7, a8";
  }
  std::ostringstream b;
  b << "rx_paged_attention<" << elem(in[0].dt) << ", " << Hq << ", " << kc.heads << ", " << kc.dim << ", " << vc.dim << ", " << kc.pages << ", " << kc.slots << ", " << B << ", " << M << ", "
    << window << ", " << (by_slot ? "true" : "false") << ", " << NT << ", " << stretches << ", " << HW << ", "
    << (once ? "true" : "false") << ", " << (dies ? "true" : "false") << ", " << (vector ? "true" : "false") << ", " << std::max<int64_t>(1, std::min<int64_t>(4, 4096 / (HW * GT * vc.dim))) << ">(a0, a1, a2, a3, a4, a5, " << (lse ? "a6" : "(float*)0") << ", " << shared << ", "
    << flt(scale * 1.4426950408889634) << ");";
  OperatorKernel k = kernel(s, "paged_attention", 256, args, (int)args.size() - 5, b.str(), waves);
  k.grid[0] = (unsigned)(B ? grid : 0);
  k.bytes = 2.0 * (double)in[0].bytes();   // (and what the lengths make of the caches)
  p.kernels.push_back(k);
  return p;
}

// ------------------------------------------------------------------ token log probabilities
void check_logprobs(const Checker& c) {
  const TType &x = c.s.in[0], &t = c.s.in[1];
  const auto& out = c.s.out;
  c.settings({"top"});
  const int64_t top = c.integer("top", 0);
  c.floats(x, "the logits");
  c.ints(t, "the targets");
  c.require(x.rank() >= 1 && x.dims.back() >= 1 && x.dims.back() <= kMaxRow, "the logits need a vocabulary: " + x.str());
  c.dims(t, without_last(x), "the targets");
  c.require(t.numel() <= kMaxRow, "too many tokens");
  c.require(top >= 0 && top <= kMaxTop && top <= x.dims.back(), "top must lie between 0 and the vocabulary's size, and be at most " + num(kMaxTop) + ", got " + num(top));
  c.require(out.size() == (top ? 5u : 3u), top ? "five results are expected with top alternatives" : "three results are expected without top alternatives");
  for (int r = 0; r < 3; ++r) {
    c.f32(out[r], "a result");
    c.dims(out[r], t.dims, "a result");
  }
  if (top) {
    std::vector<int64_t> d = t.dims;
    d.push_back(top);
    c.f32(out[3], "the top log probabilities");
    c.dims(out[3], d, "the top log probabilities");
    c.require(out[4].dt == DT::I32, "the top indices must be i32");
    c.dims(out[4], d, "the top indices");
  }
}
OperatorPlan plan_logprobs(const OperatorSpec& s) {
  const Checker c{s};
  const int64_t V = s.in[0].dims.back(), T = s.in[1].numel(), top = c.integer("top", 0);
  const int64_t vec = 16 / info(s.in[0].dt).size, vectors = (V + vec - 1) / vec + (V % vec ? 1 : 0);
  // few rows: in segments, so that every compute unit has a workgroup, of at least one round of a workgroup's loads (32 rows of 32000: 2 segments 10.9 us, 4: 10.5, 7: 11.3)
  const int64_t split = T == 0 ? 1 : std::max<int64_t>(1, std::min<int64_t>({64, (512 + T - 1) / T, vectors / 1024}));
  OperatorPlan p;
  std::vector<std::pair<OperatorArg, std::string>> args{{operand(0), st(s.in[0])}, {operand(1), st(s.in[1])}};
  for (size_t r = 0; r < s.out.size(); ++r) args.push_back({result((int)r), st(s.out[r])});
  std::string call = "rx_token_logprobs<" + std::string(elem(s.in[0].dt)) + ", " + num(V) + ", " + num(top) + ", " + num(T) + ", " + num(split) + ">(a0, a1, a2, a3, a4, " +
                     (top ? "a5, a6, " : "(float*)0, (int*)0, ");
  if (split > 1) {
    p.scratch = {T * split * 12, T * split * std::max<int64_t>(top, 1) * 8};
    p.counters = T;
    call += "a" + num((int64_t)args.size()) + ", a" + num((int64_t)args.size() + 1) + ", a" + num((int64_t)args.size() + 2) + ");";
    args.push_back({scratch(0), "float"});
    args.push_back({scratch(1), "rx_u64"});
    args.push_back({counters(), "int"});
  } else {
    call += "(float*)0, (rx_u64*)0, (int*)0);";
  }
  OperatorKernel k = kernel(s, "token_logprobs", 256, args, (int)args.size() - 2, call, split == 1 ? 6 : 0);   // six: 183 us, the compiler's five 194, eight 188 (4096 x 131072)
  k.grid[0] = (unsigned)std::min<int64_t>(T * split, kMaxGrid);
  k.bytes = (double)(s.in[0].bytes() + s.in[1].bytes());
  for (auto& t : s.out) k.bytes += (double)t.bytes();
  p.kernels.push_back(k);
  return p;
}

void check_logprobs_grad(const Checker& c) {
  const auto& in = c.s.in;
  c.settings({});
  c.floats(in[0], "the logits");
  c.ints(in[1], "the targets");
  c.require(in[0].rank() >= 1 && in[0].dims.back() >= 1 && in[0].dims.back() <= kMaxRow, "the logits need a vocabulary: " + in[0].str());
  c.dims(in[1], without_last(in[0]), "the targets");
  c.require(in[1].numel() <= kMaxRow, "too many tokens");
  for (int i = 2; i < 6; ++i) {
    c.f32(in[i], i == 2 ? "lse" : i == 3 ? "entropy" : i == 4 ? "d_logprob" : "d_entropy");
    c.dims(in[i], in[1].dims, i == 2 ? "lse" : i == 3 ? "entropy" : i == 4 ? "d_logprob" : "d_entropy");
  }
  c.same(c.s.out[0], in[0], "the logits and their gradient");
}
OperatorPlan plan_logprobs_grad(const OperatorSpec& s) {
  const int64_t V = s.in[0].dims.back(), T = s.in[1].numel();
  OperatorPlan p;
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < 6; ++i) args.push_back({operand(i), st(s.in[i])});
  args.push_back({result(0), st(s.out[0])});
  const int64_t vec = 16 / info(s.in[0].dt).size, vectors = (V + vec - 1) / vec + (V % vec ? 1 : 0);
  OperatorKernel k = kernel(s, "token_logprobs_grad", 256, args, 1,
                            std::string("rx_token_logprobs_grad<") + elem(s.in[0].dt) + ", " + num(V) + ", " + num(T) + ">(a0, a1, a2, a3, a4, a5, a6);");
  k.grid[0] = (unsigned)std::min<int64_t>(T * ((vectors + 255) / 256), kMaxGrid);
  k.bytes = 2.0 * (double)s.in[0].bytes() + 20.0 * (double)T;
  p.kernels.push_back(k);
  return p;
}

}  // namespace

bool is_operator_name(const std::string& name) {
  for (auto& o : kOperators) if (name == o.name) return true;
  return false;
}

void check_operator(const OperatorSpec& s) {
  const Checker c{s};
  for (auto& o : kOperators) {
    if (s.name != o.name) continue;
    c.require((int)s.in.size() == o.in, "expected " + num(o.in) + " operands, got " + num((int64_t)s.in.size()));
    c.require((int)s.out.size() >= o.out_min && (int)s.out.size() <= o.out_max, "wrong number of results: " + num((int64_t)s.out.size()));
  }
  for (auto& t : s.in) for (int64_t d : t.dims) c.require(d >= 0, "negative dimension");
  if (s.name == "rx.embedding") check_embedding(c);
  else if (s.name == "rx.embedding_grad") check_embedding_grad(c);
  else if (s.name == "rx.kv_append") check_append(c);
  else if (s.name == "rx.paged_attention") check_attention(c);
  else if (s.name == "rx.token_logprobs") check_logprobs(c);
  else if (s.name == "rx.token_logprobs_grad") check_logprobs_grad(c);
  else c.fail("unknown operator");
}

OperatorPlan plan_operator(const OperatorSpec& s, bool lean) {
  OperatorPlan p = s.name == "rx.embedding"         ? plan_embedding(s)
                   : s.name == "rx.embedding_grad"  ? plan_embedding_grad(s, lean)
                   : s.name == "rx.kv_append"       ? plan_append(s)
                   : s.name == "rx.paged_attention" ? plan_attention(s, lean)
                   : s.name == "rx.token_logprobs"  ? plan_logprobs(s)
                                                    : plan_logprobs_grad(s);
  // without workgroups there is nothing to compile
  p.kernels.erase(std::remove_if(p.kernels.begin(), p.kernels.end(), [](const OperatorKernel& k) { return !k.grid[0] || !k.grid[1] || !k.grid[2]; }), p.kernels.end());
  return p;
}

double operator_flops(const OperatorSpec& s, double* transcendentals) {
  *transcendentals = 0;
  if (s.name == "rx.embedding" || s.name == "rx.embedding_grad") {
    const double n = (double)s.in[1].numel() * (double)s.in[0].dims.back();
    return s.name == "rx.embedding" ? n : 2 * n;
  }
  if (s.name == "rx.kv_append") return 3.0 * 2.0 * (double)s.in[3].dims[1] * (double)(s.in[0].dims[0] * (s.in[0].dims[1] + s.in[1].dims[1]));
  if (s.name == "rx.paged_attention") {   // the longest the page table allows
    const Checker c{s};
    const Cache kc(s.in[1], c.word("layout", "slots", {"slots", "heads"}) == "slots");
    const double n = (double)(s.in[3].dims[1] * kc.slots) * (double)(s.in[0].dims[0] * s.in[0].dims[1]);
    *transcendentals = n;
    return 2.0 * n * (double)(kc.dim + s.in[2].dims[3]);
  }
  const double n = (double)s.in[0].numel();
  *transcendentals = n;
  return (s.name == "rx.token_logprobs" ? 5.0 : 6.0) * n;
}

}  // namespace rx
