// What the checks and launches of the language-model operators share (rx_lm.cpp, rx_lm_serve.cpp).
#pragma once
#include "rx_lm.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <sstream>

namespace rx {
namespace lm {

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

inline std::vector<int64_t> without_last(const TType& t) { return std::vector<int64_t>(t.dims.begin(), t.dims.end() - 1); }
inline int64_t product(const std::vector<int64_t>& d) {
  int64_t n = 1;
  for (int64_t x : d) n *= x;
  return n;
}

inline const char* elem(DT t) { return t == DT::F32 ? "rx_lm_f32" : t == DT::BF16 ? "rx_lm_bf16" : "rx_lm_f16"; }
inline std::string num(int64_t v) { return std::to_string(v); }
inline std::string flt(double v) {
  char b[40];
  snprintf(b, sizeof b, "%.9g", v);
  std::string s = b;
  if (s.find_first_of(".en") == std::string::npos) s += ".0";
  return s + "f";
}

// `body` is the call of a device function on a0, a1, ..: the kernel's parameters, of which the last `outs` are written.
// `waves`: wavefronts per SIMD that the registers have to allow (0: the compiler's choice)
inline OperatorKernel kernel(const OperatorSpec& s, const std::string& suffix, unsigned block, const std::vector<std::pair<OperatorArg, std::string>>& args, int outs,
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
inline OperatorArg operand(int i) { return {OperatorArg::Operand, i}; }
inline OperatorArg result(int i) { return {OperatorArg::Result, i}; }
inline OperatorArg scratch(int i) { return {OperatorArg::Scratch, i}; }
inline OperatorArg counters() { return {OperatorArg::Counters, 0}; }
inline std::string st(const TType& t) { return info(t.dt).stype; }

// rx_lm_serve.cpp
void check_norm(const Checker& c);
void check_norm_grad(const Checker& c);
void check_write(const Checker& c);
void check_move(const Checker& c);
void check_tree(const Checker& c);
OperatorPlan plan_norm(const OperatorSpec& s);
OperatorPlan plan_norm_grad(const OperatorSpec& s, bool lean);
OperatorPlan plan_write(const OperatorSpec& s);
OperatorPlan plan_move(const OperatorSpec& s);
OperatorPlan plan_tree(const OperatorSpec& s, bool lean);
double serve_flops(const OperatorSpec& s, double* transcendentals);

}  // namespace lm
}  // namespace rx
