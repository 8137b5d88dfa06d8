// MLIR text -> rx::Graph for the StableHLO subset of the hot path.
//
// Accepts what Reactant prints for an optimized module: pretty-printed StableHLO
// ops, generic-form ops ("stablehlo.reduce"(...) ({...})), `chlo.erf`,
// `enzymexla.math.gelu`, `func.call` (inlined), `stablehlo.optimization_barrier`
// (forwarded), attribute dictionaries on arguments (`tf.aliasing_output`, text
// sample in the reference: test/core/buffer_donation.jl:64-72) and `loc(...)`
// suffixes (test/core/compile.jl:653-661).
#include "rx_ir.h"
#include "rx_gemm.h"
#include "rx_lm.h"

#include <cmath>
#include <cstring>
#include <functional>
#include <sstream>

namespace rx {

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------
static const DTInfo kInfo[] = {
    /* I1  */ {"i1", 1, 1, "bool", "rx_u8", false, false},
    /* I8  */ {"i8", 2, 1, "rx_i8", "rx_i8", false, true},
    /* I16 */ {"i16", 3, 2, "rx_i16", "rx_i16", false, true},
    /* I32 */ {"i32", 4, 4, "rx_i32", "rx_i32", false, true},
    /* I64 */ {"i64", 5, 8, "rx_i64", "rx_i64", false, true},
    /* U8  */ {"ui8", 6, 1, "rx_u8", "rx_u8", false, false},
    /* U16 */ {"ui16", 7, 2, "rx_u16", "rx_u16", false, false},
    /* U32 */ {"ui32", 8, 4, "rx_u32", "rx_u32", false, false},
    /* U64 */ {"ui64", 9, 8, "rx_u64", "rx_u64", false, false},
    /* F16 */ {"f16", 10, 2, "float", "rx_u16", true, true},
    /* BF16*/ {"bf16", 16, 2, "float", "rx_u16", true, true},
    /* F32 */ {"f32", 11, 4, "float", "float", true, true},
    /* F64 */ {"f64", 12, 8, "double", "double", true, true},
    /* F8E4M3FN */ {"f8E4M3FN", 20, 1, "float", "rx_u8", true, true},
    /* F8E5M2 */ {"f8E5M2", 19, 1, "float", "rx_u8", true, true},
    /* INVALID */ {"?", 0, 0, "void", "void", false, false},
};

const DTInfo& info(DT t) { return kInfo[(int)t]; }

DT dt_from_mlir(const std::string& s) {
  for (int i = 0; i < (int)DT::INVALID; ++i)
    if (s == kInfo[i].mlir) return (DT)i;
  if (s == "si8") return DT::I8;
  if (s == "si16") return DT::I16;
  if (s == "si32") return DT::I32;
  if (s == "si64") return DT::I64;
  throw Error("unsupported element type '" + s + "'");
}

DT dt_from_code(int code) {
  for (int i = 0; i < (int)DT::INVALID; ++i)
    if (code == kInfo[i].code) return (DT)i;
  return DT::INVALID;
}

std::string TType::str() const {
  std::string s = "tensor<";
  for (auto d : dims) s += std::to_string(d) + "x";
  return s + info(dt).mlir + ">";
}

// ---------------------------------------------------------------------------
// host-side conversions used for constants
// ---------------------------------------------------------------------------
static uint32_t f2u(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static float u2f(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }

static uint16_t f32_to_bf16(float f) {
  uint32_t u = f2u(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  u += 0x7fffu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}
static uint8_t f32_to_f8(float f, int mbits, int bias, bool fn) {
  uint32_t u = f2u(f);
  uint8_t s = (uint8_t)((u >> 24) & 0x80u);
  float a = std::fabs(f);
  int ebits = 7 - mbits;
  int emax_field = (1 << ebits) - 1;
  uint8_t nan_code = fn ? 0x7f : (uint8_t)((emax_field << mbits) | 1 | (1 << (mbits - 1)));
  if (std::isnan(f)) return s | nan_code;
  uint8_t inf_code = fn ? 0x7f : (uint8_t)(emax_field << mbits);
  if (std::isinf(f)) return s | inf_code;
  if (a == 0) return s;
  int e;
  std::frexp(a, &e);
  e -= 1;  // a = 1.x * 2^e
  int min_e = 1 - bias;
  if (e < min_e) e = min_e;
  double q = std::ldexp(1.0, e - mbits);
  double r = std::nearbyint((double)a / q);  // ties to even (default rounding mode)
  double v = r * q;
  if (v == 0) return s;
  int e2;
  std::frexp(v, &e2);
  e2 -= 1;
  int code;
  if (v < std::ldexp(1.0, min_e)) {
    code = (int)std::nearbyint(v / std::ldexp(1.0, min_e - mbits));
  } else {
    int m = (int)std::nearbyint((v / std::ldexp(1.0, e2) - 1.0) * (1 << mbits));
    code = ((e2 + bias) << mbits) | m;
  }
  int max_code = fn ? ((emax_field << mbits) | ((1 << mbits) - 2)) : ((emax_field << mbits) - 1);
  if (code > max_code) return s | inf_code;
  return s | (uint8_t)code;
}
static uint16_t f32_to_f16(float f) {
  _Float16 h = (_Float16)f;
  uint16_t b;
  memcpy(&b, &h, 2);
  return b;
}
static float f16_to_f32(uint16_t b) {
  _Float16 h;
  memcpy(&h, &b, 2);
  return (float)h;
}
static float f8_to_f32(uint8_t b, int mbits, int bias, bool fn) {
  int ebits = 7 - mbits;
  int e = (b >> mbits) & ((1 << ebits) - 1);
  int m = b & ((1 << mbits) - 1);
  float s = (b & 0x80) ? -1.f : 1.f;
  if (fn) {
    if (e == (1 << ebits) - 1 && m == (1 << mbits) - 1) return NAN;
  } else if (e == (1 << ebits) - 1) {
    return m == 0 ? s * INFINITY : NAN;
  }
  if (e == 0) return s * std::ldexp((float)m, 1 - bias - mbits);
  return s * std::ldexp(1.0f + (float)m / (1 << mbits), e - bias);
}

static void store_scalar(DT dt, double fv, int64_t iv, bool from_int, uint8_t* out) {
  switch (dt) {
    case DT::F64: { double d = from_int ? (double)iv : fv; memcpy(out, &d, 8); break; }
    case DT::F32: { float f = from_int ? (float)iv : (float)fv; memcpy(out, &f, 4); break; }
    case DT::BF16: { uint16_t b = f32_to_bf16(from_int ? (float)iv : (float)fv); memcpy(out, &b, 2); break; }
    case DT::F16: { uint16_t b = f32_to_f16(from_int ? (float)iv : (float)fv); memcpy(out, &b, 2); break; }
    case DT::F8E4M3FN: out[0] = f32_to_f8(from_int ? (float)iv : (float)fv, 3, 7, true); break;
    case DT::F8E5M2: out[0] = f32_to_f8(from_int ? (float)iv : (float)fv, 2, 15, false); break;
    case DT::I1: out[0] = from_int ? (iv != 0) : (fv != 0); break;
    default: {
      int64_t v = from_int ? iv : (int64_t)fv;
      memcpy(out, &v, info(dt).size);  // little endian
    }
  }
}

double splat_as_double(const Node& n) {
  const uint8_t* p = n.data.data();
  switch (n.ty.dt) {
    case DT::F64: { double d; memcpy(&d, p, 8); return d; }
    case DT::F32: { float f; memcpy(&f, p, 4); return f; }
    case DT::BF16: { uint16_t b; memcpy(&b, p, 2); return u2f(((uint32_t)b) << 16); }
    case DT::F16: { uint16_t b; memcpy(&b, p, 2); return f16_to_f32(b); }
    case DT::F8E4M3FN: return f8_to_f32(p[0], 3, 7, true);
    case DT::F8E5M2: return f8_to_f32(p[0], 2, 15, false);
    default: return (double)splat_as_int(n);
  }
}

int64_t splat_as_int(const Node& n) {
  const uint8_t* p = n.data.data();
  switch (n.ty.dt) {
    case DT::I1: return p[0] != 0;
    case DT::I8: return (int8_t)p[0];
    case DT::U8: return p[0];
    case DT::I16: { int16_t v; memcpy(&v, p, 2); return v; }
    case DT::U16: { uint16_t v; memcpy(&v, p, 2); return v; }
    case DT::I32: { int32_t v; memcpy(&v, p, 4); return v; }
    case DT::U32: { uint32_t v; memcpy(&v, p, 4); return v; }
    case DT::I64: case DT::U64: { int64_t v; memcpy(&v, p, 8); return v; }
    default: return (int64_t)splat_as_double(n);
  }
}

// ---------------------------------------------------------------------------
// cursor over the text
// ---------------------------------------------------------------------------
namespace {

struct Cur {
  const char* s;
  size_t i = 0, n;
  Cur(const char* t, size_t len) : s(t), n(len) {}

  [[noreturn]] void fail(const std::string& what) const {
    size_t line = 1;
    for (size_t k = 0; k < i && k < n; ++k) line += s[k] == '\n';
    std::string ctx(s + i, std::min<size_t>(60, n - i));
    throw Error("StableHLO parse error (line " + std::to_string(line) + "): " + what + " near '" + ctx + "'");
  }
  void ws() {
    while (i < n) {
      char c = s[i];
      if (c == ' ' || c == '\t' || c == '\r' || c == '\n') ++i;
      else if (c == '/' && i + 1 < n && s[i + 1] == '/') { while (i < n && s[i] != '\n') ++i; }
      else break;
    }
  }
  char peek() { ws(); return i < n ? s[i] : '\0'; }
  bool eof() { ws(); return i >= n; }
  bool starts(const char* lit) { ws(); size_t l = strlen(lit); return i + l <= n && !strncmp(s + i, lit, l); }
  bool accept(const char* lit) {
    if (starts(lit)) { i += strlen(lit); return true; }
    return false;
  }
  void expect(const char* lit) { if (!accept(lit)) fail(std::string("expected '") + lit + "'"); }
  static bool idc(char c) { return isalnum((unsigned char)c) || c == '_' || c == '.' || c == '$'; }
  std::string ident() {
    ws();
    size_t j = i;
    if (j < n && (isalpha((unsigned char)s[j]) || s[j] == '_')) { while (j < n && idc(s[j])) ++j; }
    if (j == i) fail("expected identifier");
    std::string r(s + i, j - i);
    i = j;
    return r;
  }
  std::string ssa() {
    ws();
    if (i >= n || s[i] != '%') fail("expected SSA value");
    size_t j = i + 1;
    while (j < n && (idc(s[j]) || s[j] == '-')) ++j;
    if (j < n && s[j] == '#') { ++j; while (j < n && isdigit((unsigned char)s[j])) ++j; }
    std::string r(s + i, j - i);
    i = j;
    return r;
  }
  std::string sym() {
    ws();
    if (i >= n || s[i] != '@') fail("expected symbol");
    size_t j = i + 1;
    if (j < n && s[j] == '"') { ++j; while (j < n && s[j] != '"') ++j; ++j; }
    else while (j < n && (idc(s[j]) || s[j] == '-')) ++j;
    std::string r(s + i + 1, j - i - 1);
    i = j;
    return r;
  }
  int64_t integer() {
    ws();
    size_t j = i;
    if (j < n && (s[j] == '-' || s[j] == '+')) ++j;
    size_t d0 = j;
    while (j < n && isdigit((unsigned char)s[j])) ++j;
    if (j == d0) fail("expected integer");
    int64_t v = std::stoll(std::string(s + i, j - i));
    i = j;
    return v;
  }
  // consume "<...>" style bracketed text; returns the inside
  std::string balanced(char open, char close) {
    ws();
    if (i >= n || s[i] != open) fail(std::string("expected '") + open + "'");
    int depth = 0;
    bool in_str = false;
    for (size_t j = i; j < n; ++j) {
      char c = s[j];
      if (in_str) {
        if (c == '\\') ++j;
        else if (c == '"') in_str = false;
      } else if (c == '"') in_str = true;
      else if (c == open) ++depth;
      else if (c == close && !(close == '>' && j > 0 && s[j - 1] == '-')) {
        if (--depth == 0) {
          std::string r(s + i + 1, j - i - 1);
          i = j + 1;
          return r;
        }
      }
    }
    fail("unbalanced bracket");
  }
  // one attribute value as text: a string without its quotes, or everything up to the next comma outside of brackets
  std::string value() {
    ws();
    if (i < n && s[i] == '"') {
      size_t j = i + 1;
      while (j < n && s[j] != '"') j += s[j] == '\\' ? 2 : 1;
      if (j >= n) fail("unterminated string");
      std::string r(s + i + 1, j - i - 1);
      i = j + 1;
      return r;
    }
    int depth = 0;
    size_t j = i;
    for (; j < n; ++j) {
      const char c = s[j];
      if (c == '[' || c == '<' || c == '{' || c == '(') ++depth;
      else if (c == ']' || c == '}' || c == ')' || (c == '>' && s[j - 1] != '-')) --depth;
      else if (depth == 0 && (c == ',' || c == ':')) break;
    }
    std::string r(s + i, j - i);
    while (!r.empty() && isspace((unsigned char)r.back())) r.pop_back();
    if (r.empty()) fail("expected an attribute value");
    i = j;
    return r;
  }
  std::vector<int64_t> int_list() {
    expect("[");
    std::vector<int64_t> v;
    while (!accept("]")) { v.push_back(integer()); accept(","); }
    return v;
  }
  void skip_attr_dict() { if (peek() == '{') balanced('{', '}'); }
  void skip_loc() { if (starts("loc(")) { i += 3; balanced('(', ')'); } }

  TType type() {
    ws();
    TType t;
    if (accept("tensor")) {
      std::string in = balanced('<', '>');
      size_t p = 0;
      while (true) {
        size_t q = p;
        while (q < in.size() && isdigit((unsigned char)in[q])) ++q;
        if (q > p && q < in.size() && in[q] == 'x') {
          t.dims.push_back(std::stoll(in.substr(p, q - p)));
          p = q + 1;
        } else break;
      }
      std::string el = in.substr(p);
      size_t comma = el.find(',');
      if (comma != std::string::npos) el = el.substr(0, comma);
      while (!el.empty() && el.back() == ' ') el.pop_back();
      while (!el.empty() && el.front() == ' ') el.erase(el.begin());
      t.dt = dt_from_mlir(el);
      return t;
    }
    if (accept("!")) {  // opaque dialect type such as !stablehlo.token
      ident();
      if (peek() == '<') balanced('<', '>');
      return t;
    }
    t.dt = dt_from_mlir(ident());
    return t;
  }
  std::vector<TType> type_list_paren() {
    expect("(");
    std::vector<TType> v;
    while (!accept(")")) { v.push_back(type()); skip_attr_dict(); accept(","); }
    return v;
  }
};

struct RawOp {
  std::string name;
  std::vector<std::string> results, operands;
  std::vector<TType> tin, tout;
  std::map<std::string, std::vector<int64_t>> ia;  // integer-array attributes
  std::map<std::string, std::string> sa;            // string attributes
  std::string dense;                                // dense<> payload for constants
  std::vector<std::vector<RawOp>> regions;
  std::vector<std::pair<std::string, TType>> block_args;  // on "__block_args__"
};

struct RawFunc {
  std::string name;
  std::vector<std::pair<std::string, TType>> args;
  std::vector<std::string> arg_attrs;
  std::vector<TType> result_types;
  std::vector<RawOp> ops;
};

const char* kUnary[] = {"sine", "cosine", "tanh", "exponential", "log", "sqrt", "rsqrt", "abs", "negate", "logistic",
                        "floor", "ceil", "sign", "not", "exponential_minus_one", "log_plus_one", "round_nearest_even",
                        "round_nearest_afz", "cbrt", "tan", "is_finite", "popcnt", "count_leading_zeros", nullptr};
// the `chlo` unary ops of reference src/Ops.jl:398-436,618-640 (evaluated by the device math library)
const char* kChloUnary[] = {"chlo.erf", "chlo.erfc", "chlo.acos", "chlo.acosh", "chlo.asin", "chlo.asinh", "chlo.atan", "chlo.atanh", "chlo.cosh",
                            "chlo.sinh", "chlo.lgamma", "chlo.digamma", "chlo.erf_inv", "chlo.is_inf", "chlo.is_pos_inf", "chlo.is_neg_inf", nullptr};
const char* kBinary[] = {"add", "subtract", "multiply", "divide", "maximum", "minimum", "power", "remainder", "and", "or",
                         "xor", "atan2", "shift_left", "shift_right_logical", "shift_right_arithmetic", nullptr};
bool in_list(const char** l, const std::string& s) {
  for (; *l; ++l) if (s == *l) return true;
  return false;
}

struct P {
  Cur c;
  std::map<std::string, RawFunc> funcs;
  std::vector<std::string> func_order;
  std::string module_name;
  P(const char* t, size_t n) : c(t, n) {}

  void parse() {
    while (!c.eof()) {
      if (c.peek() == '#') { while (c.i < c.n && c.s[c.i] != '\n') ++c.i; continue; }
      if (c.accept("module")) {
        if (c.peek() == '@') module_name = c.sym();
        if (c.accept("attributes")) c.balanced('{', '}');
        c.expect("{");
        continue;
      }
      if (c.starts("func.func") || c.starts("func ")) {
        RawFunc f = func();
        func_order.push_back(f.name);
        funcs[f.name] = std::move(f);
        continue;
      }
      if (c.accept("}")) { c.skip_loc(); continue; }
      c.fail("unexpected text at module level");
    }
  }

  RawFunc func() {
    c.ident();
    for (const char* kw : {"public", "private", "nested"}) c.accept(kw);
    RawFunc f;
    f.name = c.sym();
    c.expect("(");
    while (!c.accept(")")) {
      std::string nm = c.ssa();
      c.expect(":");
      TType t = c.type();
      std::string attrs;
      if (c.peek() == '{') attrs = c.balanced('{', '}');
      c.skip_loc();
      f.args.push_back({nm, t});
      f.arg_attrs.push_back(attrs);
      c.accept(",");
    }
    if (c.accept("->")) {
      if (c.peek() == '(') f.result_types = c.type_list_paren();
      else f.result_types = {c.type()};
    }
    if (c.accept("attributes")) c.balanced('{', '}');
    c.expect("{");
    f.ops = block();
    c.skip_loc();
    return f;
  }

  std::vector<RawOp> block() {
    std::vector<RawOp> ops;
    while (true) {
      if (c.accept("}")) return ops;
      if (c.peek() == '^') {
        ++c.i;
        while (c.i < c.n && Cur::idc(c.s[c.i])) ++c.i;
        RawOp lab;
        lab.name = "__block_args__";
        if (c.peek() == '(') {
          c.expect("(");
          while (!c.accept(")")) {
            std::string nm = c.ssa();
            c.expect(":");
            TType t = c.type();
            c.skip_loc();
            lab.block_args.push_back({nm, t});
            c.accept(",");
          }
        }
        c.expect(":");
        ops.push_back(std::move(lab));
        continue;
      }
      if (c.eof()) c.fail("unterminated block");
      ops.push_back(op());
    }
  }

  void fn_type(RawOp& o) {
    if (c.peek() == '(') {
      o.tin = c.type_list_paren();
      c.expect("->");
      if (c.peek() == '(') o.tout = c.type_list_paren();
      else o.tout = {c.type()};
    } else {
      TType t = c.type();
      if (c.accept("->")) { o.tin = {t}; o.tout = {c.type()}; }
      else { o.tin = {t}; o.tout = {t}; }
    }
  }

  RawOp op() {
    std::vector<std::string> results;
    if (c.peek() == '%') {
      while (true) {
        std::string r = c.ssa();
        if (c.accept(":")) {
          int64_t k = c.integer();
          for (int64_t q = 0; q < k; ++q) results.push_back(r + "#" + std::to_string(q));
        } else results.push_back(r);
        if (!c.accept(",")) break;
      }
      c.expect("=");
    }
    RawOp o;
    if (c.peek() == '"') o = generic_op();
    else o = pretty_op(c.ident());
    o.results = results;
    c.skip_loc();
    return o;
  }

  // pull the attributes this subset needs out of a generic attribute dictionary
  static void scan_int_array(const std::string& in, const std::string& key, RawOp& o) {
    size_t p = 0;
    while ((p = in.find(key, p)) != std::string::npos) {
      bool left_ok = p == 0 || !(Cur::idc(in[p - 1]));
      size_t q = p + key.size();
      while (q < in.size() && in[q] == ' ') ++q;
      if (left_ok && q < in.size() && in[q] == '=') {
        ++q;
        while (q < in.size() && in[q] == ' ') ++q;
        std::vector<int64_t> v;
        bool ok = false;
        if (in.compare(q, 9, "array<i64") == 0) {
          size_t e = in.find('>', q);
          size_t colon = in.find(':', q);
          if (colon != std::string::npos && colon < e) {
            std::stringstream ss(in.substr(colon + 1, e - colon - 1));
            std::string tok;
            while (std::getline(ss, tok, ',')) {
              if (tok.find_first_of("0123456789") != std::string::npos) v.push_back(std::stoll(tok));
            }
          }
          ok = true;
        } else if (in.compare(q, 6, "dense<") == 0) {
          size_t e = in.find('>', q);
          std::string body = in.substr(q + 6, e - q - 6);
          for (auto& ch : body) if (ch == '[' || ch == ']') ch = ' ';
          std::stringstream ss(body);
          std::string tok;
          while (std::getline(ss, tok, ',')) {
            if (tok.find_first_of("0123456789") != std::string::npos) v.push_back(std::stoll(tok));
          }
          ok = true;
        } else if (in[q] == '[') {
          size_t e = in.find(']', q);
          std::stringstream ss(in.substr(q + 1, e - q - 1));
          std::string tok;
          while (std::getline(ss, tok, ',')) {
            if (tok.find_first_of("0123456789") != std::string::npos) v.push_back(std::stoll(tok));
          }
          ok = true;
        } else if (isdigit((unsigned char)in[q]) || in[q] == '-') {
          v.push_back(std::stoll(in.substr(q)));
          ok = true;
        }
        if (ok && !o.ia.count(key)) o.ia[key] = v;
      }
      p = q;
    }
  }

  void generic_attrs(const std::string& in, RawOp& o) {
    for (const char* key : {"dimensions", "broadcast_dimensions", "permutation", "start_indices", "limit_indices",
                            "strides", "edge_padding_low", "edge_padding_high", "interior_padding", "slice_sizes",
                            "dimension", "iota_dimension", "lhs_batching_dimensions", "rhs_batching_dimensions",
                            "lhs_contracting_dimensions", "rhs_contracting_dimensions", "window_dimensions",
                            "window_strides", "base_dilations", "window_dilations", "lhs_dilation", "rhs_dilation",
                            "padding", "feature_group_count", "batch_group_count", "feature_index", "offset_dims",
                            "collapsed_slice_dims", "operand_batching_dims", "start_indices_batching_dims", "start_index_map",
                            "index_vector_dim", "update_window_dims", "inserted_window_dims", "input_batching_dims",
                            "scatter_indices_batching_dims", "scatter_dims_to_operand_dims"})
      scan_int_array(in, key, o);
    {
      size_t q = in.find("#stablehlo.conv<");
      if (q != std::string::npos) {
        size_t arrow = in.find("->", q);
        size_t e = arrow == std::string::npos ? arrow : in.find(']', arrow);
        if (e != std::string::npos) o.sa["dim_numbers"] = in.substr(q + 16, e + 1 - (q + 16));
      }
      q = in.find("epsilon");
      if (q != std::string::npos) {
        size_t e1 = in.find('=', q);
        if (e1 != std::string::npos) {
          ++e1;
          while (e1 < in.size() && in[e1] == ' ') ++e1;
          size_t e2 = e1;
          while (e2 < in.size() && (isalnum((unsigned char)in[e2]) || in[e2] == '.' || in[e2] == '-' || in[e2] == '+')) ++e2;
          o.sa["epsilon"] = in.substr(e1, e2 - e1);
        }
      }
      q = in.find("window_reversal");
      if (q != std::string::npos) {
        size_t e = in.find('>', q);
        const std::string body = in.substr(q, e == std::string::npos ? std::string::npos : e - q);
        std::vector<int64_t> v;
        for (size_t k = 0; k < body.size(); ++k) {
          if (body.compare(k, 4, "true") == 0) v.push_back(1);
          else if (body.compare(k, 5, "false") == 0) v.push_back(0);
        }
        o.ia["window_reversal"] = v;
      }
    }
    size_t p = in.find("comparison_direction");
    if (p != std::string::npos) {
      size_t q = in.find("comparison_direction ", p + 20);
      if (q != std::string::npos) {
        q += 21;
        size_t e = q;
        while (e < in.size() && isalpha((unsigned char)in[e])) ++e;
        o.sa["direction"] = in.substr(q, e - q);
      }
    }
    p = in.find("gelu_approximation ");
    if (p != std::string::npos) {
      size_t q = p + 19, e = q;
      while (e < in.size() && isalpha((unsigned char)in[e])) ++e;
      o.sa["approximation"] = in.substr(q, e - q);
    }
    p = in.find("value");
    if (p != std::string::npos) {
      size_t q = in.find("dense<", p);
      if (q != std::string::npos) {
        Cur cc(in.c_str() + q + 5, in.size() - q - 5);
        o.dense = cc.balanced('<', '>');
      }
    }
  }

  // the target's name and its settings: `backend_config` as a dictionary of numbers and strings
  static void custom_call_attrs(const std::string& in, RawOp& o) {
    Cur a(in.c_str(), in.size());
    while (!a.eof()) {
      const std::string key = a.ident();
      if (!a.accept("=")) { a.accept(","); continue; }   // a unit attribute
      std::string* to = key == "call_target_name" ? &o.sa["call_target_name"] : key == "backend_config" ? &o.sa["backend_config"] : nullptr;
      std::string v = a.peek() == '{' ? "{" + a.balanced('{', '}') + "}" : a.value();
      if (a.accept(":")) a.value();
      if (to) *to = v;
      a.accept(",");
    }
  }

  RawOp generic_op() {
    RawOp o;
    c.ws();
    size_t j = c.i + 1;
    while (j < c.n && c.s[j] != '"') ++j;
    o.name = std::string(c.s + c.i + 1, j - c.i - 1);
    c.i = j + 1;
    c.expect("(");
    while (!c.accept(")")) { o.operands.push_back(c.ssa()); c.accept(","); }
    if (c.starts("<{")) {
      c.accept("<");
      std::string in = c.balanced('{', '}');
      c.expect(">");
      generic_attrs(in, o);
      if (o.name == "stablehlo.custom_call") custom_call_attrs(in, o);
    }
    if (c.peek() == '(') {
      c.expect("(");
      while (true) {
        c.expect("{");
        o.regions.push_back(block());
        if (!c.accept(",")) break;
      }
      c.expect(")");
    }
    if (c.peek() == '{') {
      const std::string in = c.balanced('{', '}');
      generic_attrs(in, o);
      if (o.name == "stablehlo.custom_call") custom_call_attrs(in, o);
    }
    c.expect(":");
    fn_type(o);
    return o;
  }

  RawOp pretty_op(const std::string& full) {
    RawOp o;
    o.name = full;
    std::string sh = full;
    for (const char* pre : {"stablehlo.", "mhlo.", "func."})
      if (full.rfind(pre, 0) == 0) { sh = full.substr(strlen(pre)); o.name = "stablehlo." + sh; break; }
    if (sh == "return") {
      o.name = "return";
      if (c.peek() == '%') {
        do { o.operands.push_back(c.ssa()); } while (c.accept(","));
        c.expect(":");
        do { o.tin.push_back(c.type()); } while (c.accept(","));
      }
      return o;
    }
    if (full.rfind("chlo.", 0) == 0 || full.rfind("enzymexla.", 0) == 0) {
      o.name = full;
      o.operands.push_back(c.ssa());
      while (c.accept(",")) {
        if (c.peek() == '%') o.operands.push_back(c.ssa());
        else { std::string k = c.ident(); c.expect("="); o.sa[k] = c.ident(); }
      }
      c.skip_attr_dict();
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (in_list(kUnary, sh) || in_list(kBinary, sh)) {
      do { o.operands.push_back(c.ssa()); } while (c.accept(","));
      c.skip_attr_dict();
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "constant") {
      c.skip_attr_dict();
      c.expect("dense");
      o.dense = c.balanced('<', '>');
      c.expect(":");
      o.tout = {c.type()};
      return o;
    }
    if (sh == "convert" || sh == "reshape" || sh == "bitcast_convert") {
      o.operands.push_back(c.ssa());
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "get_dimension_size") {
      // %0 = stablehlo.get_dimension_size %arg0, dim = 1 : (tensor<..>) -> tensor<i32>
      o.operands.push_back(c.ssa());
      c.expect(",");
      c.expect("dim");
      c.expect("=");
      o.ia["dimension"] = {c.integer()};
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "while") {
      // %r:2 = stablehlo.while(%iterArg = %init0, %iterArg_0 = %init1) : t0, t1 [attributes {..}]
      //   cond { ... stablehlo.return %p : tensor<i1> } do { ... stablehlo.return %a, %b : t0, t1 }
      // (the form in the docstring of the reference's binding, src/mlir/Dialects/StableHLO.jl:4850-4861)
      std::vector<std::string> names;
      c.expect("(");
      while (!c.accept(")")) {
        names.push_back(c.ssa());
        c.expect("=");
        o.operands.push_back(c.ssa());
        c.accept(",");
      }
      if (!names.empty()) {
        c.expect(":");
        do { o.tout.push_back(c.type()); } while (c.accept(","));
      }
      if (o.tout.size() != names.size()) c.fail("while: one type per loop-carried value expected");
      o.tin = o.tout;
      for (size_t k = 0; k < names.size(); ++k) o.block_args.push_back({names[k], o.tout[k]});
      if (c.accept("attributes")) c.balanced('{', '}');
      c.expect("cond");
      c.expect("{");
      o.regions.push_back(block());
      c.expect("do");
      c.expect("{");
      o.regions.push_back(block());
      return o;
    }
    if (sh == "compare") {
      o.sa["direction"] = c.ident();
      c.expect(",");
      o.operands.push_back(c.ssa());
      c.expect(",");
      o.operands.push_back(c.ssa());
      if (c.accept(",")) o.sa["compare_type"] = c.ident();
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "select") {
      for (int k = 0; k < 3; ++k) { o.operands.push_back(c.ssa()); if (k < 2) c.expect(","); }
      c.expect(":");
      if (c.peek() == '(') fn_type(o);
      else {
        TType t1 = c.type();
        if (c.accept(",")) {
          TType t2 = c.type();
          o.tin = {t1, t2, t2};
          o.tout = {t2};
        } else {
          TType tp = t1;
          tp.dt = DT::I1;
          o.tin = {tp, t1, t1};
          o.tout = {t1};
        }
      }
      return o;
    }
    if (sh == "clamp") {
      for (int k = 0; k < 3; ++k) { o.operands.push_back(c.ssa()); if (k < 2) c.expect(","); }
      c.expect(":");
      fn_type(o);
      if (o.tin.size() == 1) o.tin = {o.tin[0], o.tin[0], o.tin[0]};
      return o;
    }
    if (sh == "broadcast_in_dim" || sh == "transpose") {
      o.operands.push_back(c.ssa());
      c.expect(",");
      c.expect("dims");
      c.expect("=");
      o.ia[sh == "transpose" ? "permutation" : "broadcast_dimensions"] = c.int_list();
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "slice") {
      o.operands.push_back(c.ssa());
      c.expect("[");
      auto &st = o.ia["start_indices"], &li = o.ia["limit_indices"], &sr = o.ia["strides"];
      while (!c.accept("]")) {
        st.push_back(c.integer());
        c.expect(":");
        li.push_back(c.integer());
        sr.push_back(c.accept(":") ? c.integer() : 1);
        c.accept(",");
      }
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "pad") {
      o.operands.push_back(c.ssa());
      c.expect(",");
      o.operands.push_back(c.ssa());
      const char* keys[3][2] = {{"low", "edge_padding_low"}, {"high", "edge_padding_high"}, {"interior", "interior_padding"}};
      for (auto& k : keys) {
        c.expect(",");
        c.expect(k[0]);
        c.expect("=");
        o.ia[k[1]] = c.int_list();
      }
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "dynamic_update_slice" || sh == "dynamic_slice") {
      o.operands.push_back(c.ssa());
      while (c.accept(",")) {
        if (c.starts("sizes")) { c.expect("sizes"); c.expect("="); o.ia["slice_sizes"] = c.int_list(); }
        else o.operands.push_back(c.ssa());
      }
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "concatenate") {
      o.operands.push_back(c.ssa());
      while (c.accept(",")) {
        if (c.starts("dim")) { c.expect("dim"); c.expect("="); o.ia["dimension"] = {c.integer()}; }
        else o.operands.push_back(c.ssa());
      }
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "reverse") {
      o.operands.push_back(c.ssa());
      c.expect(",");
      c.expect("dims");
      c.expect("=");
      o.ia["dimensions"] = c.int_list();
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "convolution") {
      // stablehlo.convolution(%lhs, %rhs) dim_numbers = [b, f, 0, 1]x[o, i, 0, 1]->[b, f, 0, 1],
      //   window = {stride = [1, 1], pad = [[0, 0], [0, 0]], lhs_dilate = [..], rhs_dilate = [..], reverse = [..]}
      //   {batch_group_count = 1 : i64, feature_group_count = 1 : i64, precision_config = [..]} : (..) -> ..
      c.expect("(");
      o.operands.push_back(c.ssa());
      c.expect(",");
      o.operands.push_back(c.ssa());
      c.expect(")");
      c.expect("dim_numbers");
      c.expect("=");
      std::string dn = "[" + c.balanced('[', ']') + "]";
      c.expect("x");
      dn += "x[" + c.balanced('[', ']') + "]";
      c.expect("->");
      dn += "->[" + c.balanced('[', ']') + "]";
      o.sa["dim_numbers"] = dn;
      c.expect(",");
      c.expect("window");
      c.expect("=");
      std::string win = c.balanced('{', '}');
      // the window dictionary uses short keys; rename them to the attribute names
      RawOp tmp;
      for (const char* key : {"stride", "lhs_dilate", "rhs_dilate"}) scan_int_array(win, key, tmp);
      if (tmp.ia.count("stride")) o.ia["window_strides"] = tmp.ia["stride"];
      if (tmp.ia.count("lhs_dilate")) o.ia["lhs_dilation"] = tmp.ia["lhs_dilate"];
      if (tmp.ia.count("rhs_dilate")) o.ia["rhs_dilation"] = tmp.ia["rhs_dilate"];
      {
        size_t q = win.find("pad");
        if (q != std::string::npos && (q == 0 || !Cur::idc(win[q - 1]))) {
          size_t b0 = win.find('[', q);
          int depth = 0;
          size_t e = b0;
          for (; e < win.size(); ++e) {
            if (win[e] == '[') ++depth;
            if (win[e] == ']' && --depth == 0) break;
          }
          std::vector<int64_t> v;
          std::string body = win.substr(b0, e - b0);
          for (auto& ch : body) if (ch == '[' || ch == ']' || ch == ',') ch = ' ';
          std::stringstream ss(body);
          int64_t x;
          while (ss >> x) v.push_back(x);
          o.ia["padding"] = v;
        }
        q = win.find("reverse");
        if (q != std::string::npos) {
          size_t e = win.find(']', q);
          const std::string body = win.substr(q, e == std::string::npos ? std::string::npos : e - q);
          std::vector<int64_t> v;
          for (size_t k = 0; k < body.size(); ++k) {
            if (body.compare(k, 4, "true") == 0) v.push_back(1);
            else if (body.compare(k, 5, "false") == 0) v.push_back(0);
          }
          o.ia["window_reversal"] = v;
        }
      }
      if (c.peek() == '{') generic_attrs(c.balanced('{', '}'), o);
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "iota") {
      c.expect("dim");
      c.expect("=");
      o.ia["iota_dimension"] = {c.integer()};
      c.expect(":");
      o.tout = {c.type()};
      return o;
    }
    if (sh == "reduce") {
      // (%x init: %c) or, for several operands, (%x init: %c), (%y init: %d)
      std::vector<std::string> ins, inits;
      do {
        c.expect("(");
        do {
          ins.push_back(c.ssa());
          c.expect("init");
          c.expect(":");
          inits.push_back(c.ssa());
        } while (c.accept(","));
        c.expect(")");
      } while (c.accept(","));
      o.operands = ins;
      o.operands.insert(o.operands.end(), inits.begin(), inits.end());
      if (c.accept("applies")) {
        std::string body = c.ident();
        size_t dot = body.rfind('.');
        o.sa["body"] = dot == std::string::npos ? body : body.substr(dot + 1);
        c.expect("across");
        c.expect("dimensions");
        c.expect("=");
        o.ia["dimensions"] = c.int_list();
        c.expect(":");
        fn_type(o);
      } else {
        c.expect("across");
        c.expect("dimensions");
        c.expect("=");
        o.ia["dimensions"] = c.int_list();
        c.expect(":");
        fn_type(o);
        c.expect("reducer");
        RawOp lab;
        lab.name = "__block_args__";
        // one (lhs, rhs) group per reduced operand; the region's arguments are all lhs, then all rhs
        std::vector<std::pair<std::string, TType>> lhs, rhs;
        while (c.accept("(")) {
          std::vector<std::pair<std::string, TType>> grp;
          while (!c.accept(")")) {
            std::string nm = c.ssa();
            c.expect(":");
            TType t = c.type();
            c.skip_loc();
            grp.push_back({nm, t});
            c.accept(",");
          }
          if (grp.size() != 2) throw Error("StableHLO import: reducer group must name two arguments");
          lhs.push_back(grp[0]);
          rhs.push_back(grp[1]);
        }
        lab.block_args = lhs;
        lab.block_args.insert(lab.block_args.end(), rhs.begin(), rhs.end());
        c.expect("{");
        std::vector<RawOp> region;
        region.push_back(std::move(lab));
        auto rest = block();
        for (auto& r : rest) region.push_back(std::move(r));
        o.regions.push_back(std::move(region));
      }
      return o;
    }
    if (sh == "dot_general" || sh == "dot") {
      o.operands.push_back(c.ssa());
      c.expect(",");
      o.operands.push_back(c.ssa());
      for (const char* k : {"lhs_batching_dimensions", "rhs_batching_dimensions", "lhs_contracting_dimensions",
                            "rhs_contracting_dimensions"})
        o.ia[k] = {};
      while (c.accept(",")) {
        std::string key = c.ident();
        c.expect("=");
        if (key == "batching_dims" || key == "contracting_dims") {
          auto l = c.int_list();
          c.expect("x");
          auto r = c.int_list();
          std::string fullk = key == "batching_dims" ? "batching_dimensions" : "contracting_dimensions";
          o.ia["lhs_" + fullk] = l;
          o.ia["rhs_" + fullk] = r;
        } else if (key == "precision") o.sa["precision"] = c.balanced('[', ']');
        else if (key == "algorithm") o.sa["algorithm"] = c.balanced('<', '>');
        else c.fail("unknown dot_general attribute " + key);
      }
      c.skip_attr_dict();
      c.expect(":");
      fn_type(o);
      if (sh == "dot") {
        o.ia["lhs_contracting_dimensions"] = {(int64_t)o.tin[0].dims.size() - 1};
        o.ia["rhs_contracting_dimensions"] = {0};
        o.name = "stablehlo.dot_general";
      }
      return o;
    }
    if (sh == "optimization_barrier") {
      if (c.peek() == '%') {
        do { o.operands.push_back(c.ssa()); } while (c.accept(","));
        c.expect(":");
        do { o.tout.push_back(c.type()); } while (c.accept(","));
      }
      return o;
    }
    if (sh == "custom_call") {
      // %0:2 = stablehlo.custom_call @target(%a, %b) {backend_config = {key = value, ..}, ..} : (types) -> (types)
      o.sa["call_target_name"] = c.sym();
      c.expect("(");
      while (!c.accept(")")) { o.operands.push_back(c.ssa()); c.accept(","); }
      if (c.peek() == '{') custom_call_attrs(c.balanced('{', '}'), o);
      c.expect(":");
      fn_type(o);
      return o;
    }
    if (sh == "call") {
      o.name = "call";
      o.sa["callee"] = c.sym();
      c.expect("(");
      while (!c.accept(")")) { o.operands.push_back(c.ssa()); c.accept(","); }
      c.expect(":");
      fn_type(o);
      return o;
    }
    c.fail("unsupported operation '" + full + "'");
  }
};

// dense<> payload -> bytes in storage format
void fill_constant(Node& n, const std::string& payload_in, const std::function<void(const std::string&)>& fail) {
  std::string pl = payload_in;
  while (!pl.empty() && isspace((unsigned char)pl.front())) pl.erase(pl.begin());
  while (!pl.empty() && isspace((unsigned char)pl.back())) pl.pop_back();
  const int sz = info(n.ty.dt).size;
  const int64_t numel = n.ty.numel();
  if (!pl.empty() && pl[0] == '"') {  // hex blob
    std::string hex = pl.substr(1, pl.size() - 2);
    if (hex.rfind("0x", 0) != 0) fail("dense string payload is not hex");
    hex = hex.substr(2);
    std::vector<uint8_t> raw(hex.size() / 2);
    for (size_t k = 0; k < raw.size(); ++k) raw[k] = (uint8_t)std::stoi(hex.substr(2 * k, 2), nullptr, 16);
    if ((int64_t)raw.size() == sz && numel != 1) { n.splat = true; n.data = raw; }
    else if ((int64_t)raw.size() == numel * sz) { n.splat = numel == 1; n.data = raw; }
    else fail("dense hex payload has the wrong size");
    return;
  }
  std::vector<std::string> toks;
  std::string cur;
  for (char ch : pl) {
    if (ch == '[' || ch == ']' || ch == ',' || isspace((unsigned char)ch)) {
      if (!cur.empty()) { toks.push_back(cur); cur.clear(); }
    } else cur += ch;
  }
  if (!cur.empty()) toks.push_back(cur);
  if (toks.empty()) {
    if (numel == 0) { n.splat = false; return; }
    fail("empty dense payload");
  }
  auto put = [&](const std::string& t, uint8_t* out) {
    if (t == "true") { store_scalar(n.ty.dt, 1, 1, true, out); return; }
    if (t == "false") { store_scalar(n.ty.dt, 0, 0, true, out); return; }
    bool neg = t[0] == '-';
    std::string u = (t[0] == '-' || t[0] == '+') ? t.substr(1) : t;
    if (u.rfind("0x", 0) == 0 || u.rfind("0X", 0) == 0) {
      uint64_t bits = std::stoull(u, nullptr, 16);
      if (is_float(n.ty.dt)) { memcpy(out, &bits, sz); return; }  // bit pattern
      int64_t v = (int64_t)bits;
      store_scalar(n.ty.dt, 0, neg ? -v : v, true, out);
      return;
    }
    if (is_float(n.ty.dt)) {
      double d = (u == "inf") ? INFINITY : (u == "nan" ? NAN : std::stod(u));
      if (n.ty.dt == DT::F64) { d = neg ? -d : d; memcpy(out, &d, 8); return; }
      // decimal text -> f32 directly, then to the narrow type
      float f = (u == "inf") ? INFINITY : (u == "nan" ? NAN : std::stof(u));
      store_scalar(n.ty.dt, neg ? -f : f, 0, false, out);
      return;
    }
    if (n.ty.dt == DT::U64) { uint64_t v = std::stoull(u); memcpy(out, &v, 8); return; }
    int64_t v = std::stoll(u);
    store_scalar(n.ty.dt, 0, neg ? -v : v, true, out);
  };
  if (toks.size() == 1) {
    n.splat = true;
    n.data.resize(sz);
    put(toks[0], n.data.data());
    return;
  }
  if ((int64_t)toks.size() != numel) fail("dense payload element count does not match the type");
  n.splat = false;
  n.data.resize(numel * sz);
  for (int64_t k = 0; k < numel; ++k) put(toks[k], n.data.data() + k * sz);
}

struct Builder {
  P& p;
  Graph g;
  SplitConvs split_convs = kSplitShared;
  explicit Builder(P& pp) : p(pp) {}
  [[noreturn]] static void fail(const std::string& m) { throw Error("StableHLO import: " + m); }

  static Red body_kind(const RawOp& o) {
    std::string b;
    if (o.sa.count("body")) b = o.sa.at("body");
    else {
      if (o.regions.empty()) fail("reduce without a body");
      int cnt = 0;
      for (auto& r : o.regions[0]) {
        if (r.name == "__block_args__" || r.name == "return") continue;
        ++cnt;
        b = r.name.substr(r.name.rfind('.') + 1);
      }
      if (cnt != 1) fail("reduce body must be a single monoid operation");
    }
    if (b == "add") return Red::Add;
    if (b == "multiply") return Red::Mul;
    if (b == "maximum") return Red::Max;
    if (b == "minimum") return Red::Min;
    if (b == "and") return Red::And;
    if (b == "or") return Red::Or;
    fail("unsupported reduce body '" + b + "'");
  }

  std::vector<int> inline_func(const RawFunc& f, const std::vector<int>& args, int depth) {
    if (depth > 16) fail("call depth exceeded");
    if (args.size() != f.args.size()) fail("call to @" + f.name + " with wrong argument count");
    std::map<std::string, int> env;
    for (size_t k = 0; k < args.size(); ++k) env[f.args[k].first] = args[k];
    return run_block(f.ops, env, depth);
  }

  std::vector<int> run_block(const std::vector<RawOp>& ops, std::map<std::string, int>& env, int depth) {
    auto look = [&](const std::string& s) -> int {
      auto it = env.find(s);
      if (it == env.end()) {
        // "%x" may refer to the single result of "%x:1" and vice versa
        auto it2 = env.find(s + "#0");
        if (it2 != env.end()) return it2->second;
        fail("use of undefined value " + s);
      }
      return it->second;
    };
    for (auto& o : ops) {
      if (o.name == "__block_args__") continue;
      std::vector<int> in;
      for (auto& s : o.operands) in.push_back(look(s));
      if (o.name == "return" || o.name == "stablehlo.return" || o.name == "func.return") return in;
      std::vector<int> outs = o.name == "stablehlo.while" ? run_while(o, in, env, depth)
                              : (o.name == "stablehlo.if" || o.name == "stablehlo.case") ? run_branches(o, in, env, depth)
                                                                                         : build(o, in, depth);
      if (outs.size() != o.results.size()) fail("result count mismatch on " + o.name);
      for (size_t k = 0; k < outs.size(); ++k) env[o.results[k]] = outs[k];
    }
    return {};
  }

  const TType& ty(int id) { return g.nodes[id].ty; }

  // ---- loops with a static trip count -------------------------------------------------------
  // `stablehlo.while` is unrolled while the module is imported: the condition region is
  // evaluated on the current loop-carried values and must fold to a constant (an induction
  // variable compared with a constant); each time it is true the body region is replayed.  This
  // is the form `@trace for` loops take (reference src/Ops.jl:2349-2460); loops whose trip count
  // depends on data are rejected.
  static constexpr int kMaxTrip = 65536;
  std::map<int, std::pair<bool, int64_t>> folded;

  static bool is_int_dt(DT t) { return !is_float(t) && t != DT::INVALID; }
  static int64_t wrap_to(DT t, int64_t v) {
    switch (t) {
      case DT::I1: return v != 0;
      case DT::I8: return (int8_t)v;
      case DT::I16: return (int16_t)v;
      case DT::I32: return (int32_t)v;
      case DT::U8: return (uint8_t)v;
      case DT::U16: return (uint16_t)v;
      case DT::U32: return (uint32_t)v;
      default: return v;
    }
  }
  static bool is_unsigned_dt(DT t) { return t == DT::U8 || t == DT::U16 || t == DT::U32 || t == DT::U64; }

  // value of a one-element integer node that depends on constants only
  bool fold_int(int id, int64_t* out) {
    auto it = folded.find(id);
    if (it != folded.end()) { *out = it->second.second; return it->second.first; }
    const Node& n = g.nodes[id];
    bool ok = false;
    int64_t v = 0;
    auto sub = [&](int k, int64_t* x) { return fold_int(n.in[k], x); };
    if (is_int_dt(n.ty.dt) && n.ty.numel() == 1) {
      int64_t a, b, c2;
      switch (n.k) {
        case OpK::Constant:
          if (n.splat || n.data.size() == (size_t)info(n.ty.dt).size) { v = splat_as_int(n); ok = true; }
          break;
        case OpK::Convert:
          if (is_int_dt(g.nodes[n.in[0]].ty.dt) && sub(0, &a)) { v = wrap_to(n.ty.dt, a); ok = true; }
          break;
        case OpK::Reshape:
        case OpK::BroadcastInDim:
          if (sub(0, &a)) { v = a; ok = true; }
          break;
        case OpK::Binary:
          if (sub(0, &a) && sub(1, &b)) {
            const bool un = is_unsigned_dt(n.ty.dt);
            ok = true;
            if (n.op == "add") v = (int64_t)((uint64_t)a + (uint64_t)b);
            else if (n.op == "subtract") v = (int64_t)((uint64_t)a - (uint64_t)b);
            else if (n.op == "multiply") v = (int64_t)((uint64_t)a * (uint64_t)b);
            else if (n.op == "minimum") v = un ? (int64_t)std::min((uint64_t)a, (uint64_t)b) : std::min(a, b);
            else if (n.op == "maximum") v = un ? (int64_t)std::max((uint64_t)a, (uint64_t)b) : std::max(a, b);
            else if (n.op == "and") v = a & b;
            else if (n.op == "or") v = a | b;
            else if (n.op == "xor") v = a ^ b;
            else ok = false;
            v = wrap_to(n.ty.dt, v);
          }
          break;
        case OpK::Unary:
          if (sub(0, &a)) {
            ok = true;
            if (n.op == "negate") v = wrap_to(n.ty.dt, (int64_t)(0 - (uint64_t)a));
            else if (n.op == "not") v = n.ty.dt == DT::I1 ? !a : wrap_to(n.ty.dt, ~a);
            else ok = false;
          }
          break;
        case OpK::Compare:
          if (is_int_dt(g.nodes[n.in[0]].ty.dt) && sub(0, &a) && sub(1, &b)) {
            const bool un = is_unsigned_dt(g.nodes[n.in[0]].ty.dt) || n.cmp_unsigned;
            const bool lt = un ? (uint64_t)a < (uint64_t)b : a < b, eq = a == b;
            ok = true;
            if (n.op == "LT") v = lt;
            else if (n.op == "LE") v = lt || eq;
            else if (n.op == "GT") v = !lt && !eq;
            else if (n.op == "GE") v = !lt;
            else if (n.op == "EQ") v = eq;
            else if (n.op == "NE") v = !eq;
            else ok = false;
          }
          break;
        case OpK::Select:
          if (sub(0, &c2) && sub(1, &a) && sub(2, &b)) { v = c2 ? a : b; ok = true; }
          break;
        default:
          break;
      }
    }
    folded[id] = {ok, v};
    *out = v;
    return ok;
  }

  // `stablehlo.if` / `stablehlo.case` (what `@trace if` prints, reference src/Ops.jl:2449-2470,2838,3198).
  // A predicate that folds to a constant selects its branch while importing.  Otherwise every
  // branch is evaluated and the results are selected element by element: regions of this op set
  // have no side effects, so the values are those of running the one branch.
  std::vector<int> run_branches(const RawOp& o, const std::vector<int>& in, const std::map<std::string, int>& outer, int depth) {
    if (depth > 16) fail(o.name + ": nesting depth exceeded");
    const bool is_if = o.name == "stablehlo.if";
    if (in.size() != 1 || ty(in[0]).numel() != 1 || ty(in[0]).rank() != 0) fail(o.name + ": expected one 0-d predicate / index operand");
    if (is_if ? (o.regions.size() != 2 || ty(in[0]).dt != DT::I1) : (o.regions.empty() || !is_int_dt(ty(in[0]).dt) || ty(in[0]).dt == DT::I1))
      fail(o.name + ": malformed regions or operand type");
    const int nbr = (int)o.regions.size();
    int64_t folded_v = 0;
    const bool is_const = fold_int(in[0], &folded_v);
    auto run_one = [&](int k) {
      std::map<std::string, int> env = outer;
      std::vector<int> r = run_block(o.regions[k], env, depth + 1);
      if (r.size() != o.tout.size()) fail(o.name + ": a branch returns " + std::to_string(r.size()) + " values for " + std::to_string(o.tout.size()) + " results");
      for (size_t q = 0; q < r.size(); ++q) if (!(ty(r[q]) == o.tout[q])) fail(o.name + ": branch result " + std::to_string(q) + " has type " + ty(r[q]).str());
      return r;
    };
    if (is_const) {
      // if: region 0 is the true branch; case: an index outside [0, n) selects the last branch
      const int k = is_if ? (folded_v ? 0 : 1) : (int)((folded_v < 0 || folded_v >= nbr) ? nbr - 1 : folded_v);
      return run_one(k);
    }
    std::vector<std::vector<int>> vals;
    for (int k = 0; k < nbr; ++k) vals.push_back(run_one(k));
    auto select_node = [&](int pred, int a, int b) {
      const TType t = ty(a);
      int p = pred;
      if (t.rank() != 0) {
        Node bc;
        bc.k = OpK::BroadcastInDim;
        bc.in = {pred};
        bc.ty = TType{DT::I1, t.dims};
        p = g.add(bc);
      }
      Node sn;
      sn.k = OpK::Select;
      sn.in = {p, a, b};
      sn.ty = t;
      return g.add(sn);
    };
    std::vector<int> out;
    for (size_t q = 0; q < o.tout.size(); ++q) {
      if (is_if) { out.push_back(select_node(in[0], vals[0][q], vals[1][q])); continue; }
      // case: start from the last branch (also the out-of-range choice), override with index == k
      int cur = vals[nbr - 1][q];
      for (int k = nbr - 2; k >= 0; --k) {
        Node c;
        c.k = OpK::Constant;
        c.splat = true;
        c.ty = ty(in[0]);
        c.data.assign((size_t)info(c.ty.dt).size, 0);
        store_scalar(c.ty.dt, (double)k, k, true, c.data.data());
        const int ci = g.add(c);
        Node eq;
        eq.k = OpK::Compare;
        eq.op = "EQ";
        eq.in = {in[0], ci};
        eq.ty = TType{DT::I1, {}};
        cur = select_node(g.add(eq), vals[k][q], cur);
      }
      out.push_back(cur);
    }
    return out;
  }

  std::vector<int> run_while(const RawOp& o, const std::vector<int>& init, const std::map<std::string, int>& outer, int depth) {
    if (depth > 16) fail("while: nesting depth exceeded");
    if (o.regions.size() != 2) fail("while: expected a condition and a body region");
    auto names_of = [&](const std::vector<RawOp>& region) {
      std::vector<std::pair<std::string, TType>> a = o.block_args;
      if (a.empty())
        for (auto& r : region)
          if (r.name == "__block_args__") { a = r.block_args; break; }
      if (a.size() != init.size()) fail("while: " + std::to_string(a.size()) + " region arguments for " + std::to_string(init.size()) + " loop-carried values");
      return a;
    };
    const auto cond_args = names_of(o.regions[0]), body_args = names_of(o.regions[1]);
    for (size_t k = 0; k < init.size(); ++k) {
      if (!(ty(init[k]) == cond_args[k].second)) fail("while: operand " + std::to_string(k) + " has type " + ty(init[k]).str() + ", region expects " + cond_args[k].second.str());
      if (k < o.tout.size() && !(o.tout[k] == ty(init[k]))) fail("while: result " + std::to_string(k) + " type mismatch");
    }
    std::vector<int> cur = init;
    for (int trip = 0;; ++trip) {
      if (trip > kMaxTrip) fail("while: more than " + std::to_string(kMaxTrip) + " iterations");
      std::map<std::string, int> env = outer;
      for (size_t k = 0; k < cur.size(); ++k) env[cond_args[k].first] = cur[k];
      std::vector<int> pred = run_block(o.regions[0], env, depth + 1);
      if (pred.size() != 1 || ty(pred[0]).dt != DT::I1 || ty(pred[0]).numel() != 1) fail("while: the condition must return one tensor<i1>");
      int64_t p = 0;
      if (!fold_int(pred[0], &p))
        fail("while: the condition does not fold to a constant; only loops with a static trip count are supported");
      if (!p) return cur;
      env = outer;
      for (size_t k = 0; k < cur.size(); ++k) env[body_args[k].first] = cur[k];
      std::vector<int> next = run_block(o.regions[1], env, depth + 1);
      if (next.size() != cur.size()) fail("while: the body returns " + std::to_string(next.size()) + " values for " + std::to_string(cur.size()) + " loop-carried ones");
      for (size_t k = 0; k < cur.size(); ++k)
        if (!(ty(next[k]) == ty(cur[k]))) fail("while: the body changes the type of loop-carried value " + std::to_string(k));
      cur = next;
    }
  }

  // An unrolled loop that reads `a[i]` (dynamic_slice at the loop counter) leaves one dynamic_slice per
  // trip, alike but for the folded start.  Written into the kernel text the starts would make every
  // trip's kernel a different one (hundreds of compilations for a time loop); kept as 0-d constants in
  // memory, the trips share one kernel text that reads its start from its own 8-byte buffer.
  void keep_loop_slice_starts_in_memory() {
    std::map<std::pair<int, std::vector<int64_t>>, std::vector<int>> groups;
    std::vector<int> other_uses(g.nodes.size(), 0);
    for (int r : g.results) other_uses[r]++;
    for (const Node& n : g.nodes) {
      bool all_const = n.k == OpK::DynamicSlice;
      for (size_t k = 0; k < n.in.size(); ++k) {
        if (n.k == OpK::DynamicSlice && k >= 1) all_const = all_const && g.nodes[n.in[k]].k == OpK::Constant && g.nodes[n.in[k]].ty.rank() == 0;
        else other_uses[n.in[k]]++;
      }
      if (all_const) groups[{n.in[0], n.a0}].push_back(n.id);
    }
    for (auto& kv : groups) {
      if (kv.second.size() < 8) continue;
      for (int id : kv.second)
        for (size_t k = 1; k < g.nodes[id].in.size(); ++k) {
          Node& c = g.nodes[g.nodes[id].in[k]];
          if (other_uses[c.id] == 0 && c.data.size() == (size_t)info(c.ty.dt).size) c.splat = false;
        }
    }
  }

  // one-element integer values that depend on constants only become constants (loop counters
  // after unrolling; start indices of dynamic slices must be constants when kernels are planned)
  void fold_scalar_constants() {
    for (size_t id = 0; id < g.nodes.size(); ++id) {
      Node& n = g.nodes[id];
      if (n.k == OpK::Constant || n.k == OpK::Param || n.in.empty()) continue;
      if (!is_int_dt(n.ty.dt) || n.ty.numel() != 1) continue;
      int64_t v;
      if (!fold_int((int)id, &v)) continue;
      n.k = OpK::Constant;
      n.op.clear();
      n.in.clear();
      n.a0.clear(); n.a1.clear(); n.a2.clear(); n.a3.clear();
      n.splat = true;
      n.data.assign(info(n.ty.dt).size, 0);
      store_scalar(n.ty.dt, (double)v, v, true, n.data.data());
    }
  }

  void check_same(const TType& a, const TType& b, const std::string& what) {
    if (!(a == b)) fail(what + ": type mismatch " + a.str() + " vs " + b.str());
  }

  int add_node(OpK k, const TType& t, std::vector<int> in) {
    Node n;
    n.k = k;
    n.ty = t;
    n.in = std::move(in);
    return g.add(n);
  }
  int zero_of(DT dt) {
    Node z;
    z.k = OpK::Constant;
    z.splat = true;
    z.ty = TType{dt, {}};
    z.data.assign((size_t)info(dt).size, 0);
    return g.add(z);
  }
  // the strided window view of `x`: [w_0..w_{r-1}, o_0..o_{r-1}]
  int window_view(int x, const std::vector<int64_t>& w, const std::vector<int64_t>& st, const std::vector<int64_t>& dl,
                  const std::string& what) {
    const TType& t = ty(x);
    const int r = t.rank();
    Node n;
    n.k = OpK::Window;
    n.in = {x};
    n.a0 = w; n.a1 = st; n.a2 = dl;
    n.ty.dt = t.dt;
    n.ty.dims = w;
    for (int d = 0; d < r; ++d) {
      if (w[d] < 1 || st[d] < 1 || dl[d] < 1) fail(what + ": window sizes, strides and dilations must be positive");
      const int64_t span = (w[d] - 1) * dl[d] + 1;
      n.ty.dims.push_back(t.dims[d] < span ? 0 : (t.dims[d] - span) / st[d] + 1);
    }
    return g.add(n);
  }

  // reduce_window (reference src/Ops.jl:3967-4011).  Pooling (ext/ReactantNNlibExt/Ops.jl:1-32)
  // becomes pad + window view + reduce over the window dims; the form cumsum/cumprod build
  // (src/TracedRArray.jl:1086-1108: the window spans one whole dimension, padded by its length
  // minus one on one side) becomes a prefix scan.
  int build_reduce_window(const RawOp& o, int x, int init, const TType& out) {
    const TType xt = ty(x);
    const int r = xt.rank();
    if (ty(init).rank() != 0 || ty(init).dt != xt.dt || out.dt != xt.dt) fail("reduce_window: operand, init and result element types must match");
    const Red red = body_kind(o);
    auto get = [&](const char* key, int64_t dflt) {
      std::vector<int64_t> v = o.ia.count(key) ? o.ia.at(key) : std::vector<int64_t>(r, dflt);
      if ((int)v.size() != r) fail(std::string("reduce_window: ") + key + " must have one entry per dimension");
      return v;
    };
    if (!o.ia.count("window_dimensions")) fail("reduce_window: window_dimensions missing");
    const auto w = get("window_dimensions", 1), st = get("window_strides", 1), bd = get("base_dilations", 1), wd = get("window_dilations", 1);
    std::vector<int64_t> pad = o.ia.count("padding") ? o.ia.at("padding") : std::vector<int64_t>(2 * r, 0);
    if (pad.size() == 1) pad.assign(2 * r, pad[0]);
    if ((int)pad.size() != 2 * r) fail("reduce_window: padding must be a (rank x 2) matrix");
    std::vector<int64_t> lo(r), hi(r), interior(r);
    bool any_pad = false;
    for (int d = 0; d < r; ++d) {
      lo[d] = pad[2 * d]; hi[d] = pad[2 * d + 1]; interior[d] = bd[d] - 1;
      if (lo[d] < 0 || hi[d] < 0 || bd[d] < 1) fail("reduce_window: negative padding is not supported");
      any_pad = any_pad || lo[d] || hi[d] || interior[d];
    }
    // prefix form
    int sd = -1, others = 0;
    for (int d = 0; d < r; ++d) {
      const bool unit = w[d] == 1 && st[d] == 1 && lo[d] == 0 && hi[d] == 0 && bd[d] == 1;
      if (unit) continue;
      ++others;
      const bool fwd = lo[d] == xt.dims[d] - 1 && hi[d] == 0, bwd = lo[d] == 0 && hi[d] == xt.dims[d] - 1;
      if (w[d] == xt.dims[d] && st[d] == 1 && wd[d] == 1 && bd[d] == 1 && (fwd || bwd) && xt.dims[d] > 1) sd = d;
    }
    if (others == 1 && sd >= 0 && xt.numel() > 0 && xt.dt != DT::I1) {
      if (!(out == xt)) fail("reduce_window: result shape mismatch");
      Node n;
      n.k = OpK::Scan;
      n.ty = xt;
      n.in = {x, init};
      n.red = red;
      n.a0 = {sd};
      n.a1 = {lo[sd] == 0 ? 1 : 0};
      return g.add(n);
    }
    int cur = x;
    if (any_pad) {
      Node pn;
      pn.k = OpK::Pad;
      pn.in = {x, init};
      pn.a0 = lo; pn.a1 = hi; pn.a2 = interior;
      pn.ty.dt = xt.dt;
      for (int d = 0; d < r; ++d) pn.ty.dims.push_back(lo[d] + hi[d] + xt.dims[d] + std::max<int64_t>(xt.dims[d] - 1, 0) * interior[d]);
      cur = g.add(pn);
    }
    const int win = window_view(cur, w, st, wd, "reduce_window");
    const TType wt = ty(win);
    if (std::vector<int64_t>(wt.dims.begin() + r, wt.dims.end()) != out.dims) fail("reduce_window: result shape mismatch");
    Node rn;
    rn.k = OpK::Reduce;
    rn.in = {win, init};
    rn.red = red;
    for (int d = 0; d < r; ++d) rn.a0.push_back(d);
    rn.ty = out;
    return g.add(rn);
  }

  // select_and_scatter in the form the gradient of max / min pooling takes (select: one compare of
  // the two values, scatter: add).  Per window: the position of the extreme (the first one in
  // row-major window order for GE / LE, the last for GT / LT) from an index reduction over the
  // window view, turned into operand coordinates; then a scatter-add of `source` into an operand-shaped
  // array of `init`.  Padding never wins against data (it holds -inf / +inf); a window made of padding
  // only lands outside the operand and is dropped by the scatter.
  int build_select_and_scatter(const RawOp& o, int x, int src, int init, const TType& out) {
    const char* what = "select_and_scatter: only the pooling-gradient form is supported (select = one GE / GT / LE / LT compare, scatter = add)";
    const TType xt = ty(x), st_ = ty(src);
    const int r = xt.rank();
    if (!(out == xt) || !is_float(xt.dt) || is_narrow_float(xt.dt) || st_.dt != xt.dt || ty(init).rank() != 0 || r < 1) fail(what);
    if (o.regions.size() != 2) fail(what);
    auto body_of = [&](const std::vector<RawOp>& region, std::string* a, std::string* b) {
      if (region.size() != 3 || region[0].name != "__block_args__" || region[0].block_args.size() != 2) fail(what);
      *a = region[0].block_args[0].first; *b = region[0].block_args[1].first;
      const RawOp& ret = region[2];
      if (region[1].results.size() != 1 || ret.operands.size() != 1 || ret.operands[0] != region[1].results[0]) fail(what);
      return &region[1];
    };
    std::string a, b;
    const RawOp* cmp = body_of(o.regions[0], &a, &b);
    if (cmp->name.substr(cmp->name.rfind('.') + 1) != "compare" || cmp->operands.size() != 2 || cmp->operands[0] != a || cmp->operands[1] != b) fail(what);
    const std::string dir = cmp->sa.count("direction") ? cmp->sa.at("direction") : "";
    const bool is_max = dir == "GE" || dir == "GT", is_min = dir == "LE" || dir == "LT";
    if (!is_max && !is_min) fail(what);
    const bool first = dir == "GE" || dir == "LE";
    const RawOp* add = body_of(o.regions[1], &a, &b);
    if (add->name.substr(add->name.rfind('.') + 1) != "add" || add->operands.size() != 2 ||
        !((add->operands[0] == a && add->operands[1] == b) || (add->operands[0] == b && add->operands[1] == a))) fail(what);
    auto get = [&](const char* key, int64_t dflt) {
      std::vector<int64_t> v = o.ia.count(key) ? o.ia.at(key) : std::vector<int64_t>(r, dflt);
      if ((int)v.size() != r) fail(std::string("select_and_scatter: ") + key + " must have one entry per dimension");
      return v;
    };
    if (!o.ia.count("window_dimensions")) fail("select_and_scatter: window_dimensions missing");
    const auto w = get("window_dimensions", 1), st = get("window_strides", 1);
    std::vector<int64_t> pad = o.ia.count("padding") ? o.ia.at("padding") : std::vector<int64_t>(2 * r, 0);
    if (pad.size() == 1) pad.assign(2 * r, pad[0]);
    if ((int)pad.size() != 2 * r) fail("select_and_scatter: padding must be a (rank x 2) matrix");
    std::vector<int64_t> lo(r), hi(r), zeros(r, 0), ones(r, 1);
    bool any_pad = false;
    for (int d = 0; d < r; ++d) {
      lo[d] = pad[2 * d]; hi[d] = pad[2 * d + 1];
      if (lo[d] < 0 || hi[d] < 0) fail("select_and_scatter: negative padding is not supported");
      any_pad = any_pad || lo[d] || hi[d];
    }
    int cur = x;
    if (any_pad) {
      Node c;
      c.k = OpK::Constant;
      c.splat = true;
      c.ty = TType{xt.dt, {}};
      c.data.assign((size_t)info(xt.dt).size, 0);
      store_scalar(xt.dt, is_max ? -INFINITY : INFINITY, 0, false, c.data.data());
      const int pv = g.add(c);
      Node pn;
      pn.k = OpK::Pad;
      pn.in = {x, pv};
      pn.a0 = lo; pn.a1 = hi; pn.a2 = zeros;
      pn.ty.dt = xt.dt;
      for (int d = 0; d < r; ++d) pn.ty.dims.push_back(lo[d] + hi[d] + xt.dims[d]);
      cur = g.add(pn);
    }
    const int win = window_view(cur, w, st, ones, "select_and_scatter");       // [w.., o..]
    const TType wt = ty(win);
    const std::vector<int64_t> odims(wt.dims.begin() + r, wt.dims.end());
    if (odims != st_.dims) fail("select_and_scatter: source shape does not match the windows");
    int64_t wn = 1;
    for (int d = 0; d < r; ++d) wn *= w[d];
    std::vector<int64_t> fdims{wn};
    fdims.insert(fdims.end(), odims.begin(), odims.end());
    const TType ft{xt.dt, fdims}, it{DT::I64, fdims}, ot{DT::I64, odims};
    const int flat = add_node(OpK::Reshape, ft, {win});
    // the extreme of every window, and the flat window offset that holds it
    Node m;
    m.k = OpK::Reduce;
    m.red = is_max ? Red::Max : Red::Min;
    {
      Node c;
      c.k = OpK::Constant;
      c.splat = true;
      c.ty = TType{xt.dt, {}};
      c.data.assign((size_t)info(xt.dt).size, 0);
      store_scalar(xt.dt, is_max ? -INFINITY : INFINITY, 0, false, c.data.data());
      m.in = {flat, g.add(c)};
    }
    m.a0 = {0};
    m.ty = TType{xt.dt, odims};
    const int mv = g.add(m);
    Node mb;
    mb.k = OpK::BroadcastInDim;
    mb.in = {mv};
    mb.ty = ft;
    for (int d = 0; d < r; ++d) mb.a0.push_back(d + 1);
    const int mbv = g.add(mb);
    Node eq;
    eq.k = OpK::Compare;
    eq.op = "EQ";
    eq.in = {flat, mbv};
    eq.ty = TType{DT::I1, fdims};
    const int eqv = g.add(eq);
    Node io;
    io.k = OpK::Iota;
    io.ty = it;
    io.a0 = {0};
    const int iov = g.add(io);
    const int limv = splat_of(it, first ? (double)wn : -1.0);
    Node sel;
    sel.k = OpK::Select;
    sel.in = {eqv, iov, limv};
    sel.ty = it;
    const int selv = g.add(sel);
    Node jr;
    jr.k = OpK::Reduce;
    jr.red = first ? Red::Min : Red::Max;
    jr.in = {selv, splat_of(TType{DT::I64, {}}, first ? (double)wn : -1.0)};
    jr.a0 = {0};
    jr.ty = ot;
    const int jv = g.add(jr);
    // operand coordinates of the selected element: o_d * stride_d + j_d - lo_d, stacked along a new last dim
    std::vector<int64_t> idims = odims;
    idims.push_back(1);
    std::vector<int> parts;
    int64_t inner = wn;
    for (int d = 0; d < r; ++d) {
      inner /= w[d];
      int jd = binary_node("divide", jv, splat_of(ot, (double)inner));
      jd = binary_node("remainder", jd, splat_of(ot, (double)w[d]));
      Node od;
      od.k = OpK::Iota;
      od.ty = ot;
      od.a0 = {d};
      int pos = binary_node("multiply", g.add(od), splat_of(ot, (double)st[d]));
      pos = binary_node("add", pos, jd);
      pos = binary_node("subtract", pos, splat_of(ot, (double)lo[d]));
      parts.push_back(add_node(OpK::Reshape, TType{DT::I64, idims}, {pos}));
    }
    int index = parts[0];
    if (r > 1) {
      Node cc;
      cc.k = OpK::Concatenate;
      cc.in = parts;
      cc.a0 = {r};
      cc.ty = TType{DT::I64, odims};
      cc.ty.dims.push_back(r);
      index = g.add(cc);
    }
    Node ib;
    ib.k = OpK::BroadcastInDim;
    ib.in = {init};
    ib.ty = xt;
    const int base = g.add(ib);
    Node sc;
    sc.k = OpK::Scatter;
    sc.ty = xt;
    sc.in = {base, index, src};
    for (int d = 0; d < r; ++d) { sc.a1.push_back(d); sc.a2.push_back(d); }
    sc.a4 = {r};
    sc.op = "combine";
    sc.red = Red::Add;
    return g.add(sc);
  }

  int binary_node(const char* op, int a, int b) {
    Node n;
    n.k = OpK::Binary;
    n.op = op;
    n.ty = ty(a);
    n.in = {a, b};
    return g.add(n);
  }
  int splat_of(const TType& t, double v) {
    Node c;
    c.k = OpK::Constant;
    c.splat = true;
    c.ty = TType{t.dt, {}};
    c.data.assign((size_t)info(t.dt).size, 0);
    store_scalar(t.dt, v, (int64_t)v, false, c.data.data());
    const int id = g.add(c);
    if (t.rank() == 0) return id;
    Node b;
    b.k = OpK::BroadcastInDim;
    b.in = {id};
    b.ty = t;
    return g.add(b);
  }
  int feature_bcast(int v, const TType& full, int feature) {
    Node b;
    b.k = OpK::BroadcastInDim;
    b.in = {v};
    b.a0 = {feature};
    b.ty = full;
    return g.add(b);
  }
  // batch_norm_inference / batch_norm_training (reference src/Ops.jl:4012-4092), written out as the
  // specification defines them: per-feature mean and biased variance over all other dims (training),
  // then (x - mean) / sqrt(variance + epsilon) * scale + offset.
  std::vector<int> build_batch_norm(const RawOp& o, const std::vector<int>& in, bool training) {
    if (in.size() != (training ? 3u : 5u)) fail(o.name + ": wrong operand count");
    if (!o.ia.count("feature_index") || o.ia.at("feature_index").empty()) fail(o.name + ": feature_index missing");
    if (!o.sa.count("epsilon")) fail(o.name + ": epsilon missing");
    const TType xt = ty(in[0]);
    const int f = (int)o.ia.at("feature_index")[0];
    if (!is_float(xt.dt) || f < 0 || f >= xt.rank()) fail(o.name + ": float operand and a valid feature_index expected");
    const TType ft{xt.dt, {xt.dims[f]}};
    for (size_t k = 1; k < in.size(); ++k) if (!(ty(in[k]) == ft)) fail(o.name + ": per-feature operands must be " + ft.str());
    if (o.tout.empty() || !(o.tout[0] == xt)) fail(o.name + ": result type mismatch");
    double eps = 0;
    try { eps = std::stod(o.sa.at("epsilon")); } catch (...) { fail(o.name + ": malformed epsilon"); }
    int mean, var;
    if (training) {
      std::vector<int64_t> rdims;
      double count = 1;
      for (int d = 0; d < xt.rank(); ++d) if (d != f) { rdims.push_back(d); count *= (double)xt.dims[d]; }
      auto feature_mean = [&](int v) {
        Node r;
        r.k = OpK::Reduce;
        r.red = Red::Add;
        r.in = {v, zero_of(xt.dt)};
        r.a0 = rdims;
        r.ty = ft;
        return binary_node("divide", g.add(r), splat_of(ft, count));
      };
      mean = feature_mean(in[0]);
      const int c = binary_node("subtract", in[0], feature_bcast(mean, xt, f));
      var = feature_mean(binary_node("multiply", c, c));
    } else {
      mean = in[3];
      var = in[4];
    }
    const int centered = binary_node("subtract", in[0], feature_bcast(mean, xt, f));
    Node sq;
    sq.k = OpK::Unary;
    sq.op = "sqrt";
    sq.ty = ft;
    sq.in = {binary_node("add", var, splat_of(ft, eps))};
    const int stddev = g.add(sq);
    const int normalized = binary_node("divide", centered, feature_bcast(stddev, xt, f));
    const int res = binary_node("add", binary_node("multiply", normalized, feature_bcast(in[1], xt, f)), feature_bcast(in[2], xt, f));
    if (training) return {res, mean, var};
    return {res};
  }

  // The reduce over (value, index) pairs that argmax / argmin / findmax / findmin print
  // (reference src/Ops.jl:1571-1596): body `c = a1 <dir> a2; return select(c, a1, a2), select(c, i1, i2)`
  // with the indices an iota along the one reduced dimension.  It becomes two monoid reductions:
  // the extreme value, then the first (non-strict comparison) or last (strict) index that holds it.
  // A slice in which no element equals the extreme (NaNs) gets the largest / smallest index value.
  std::vector<int> build_arg_reduce(const RawOp& o, const std::vector<int>& in) {
    const char* what = "reduce over two operands: only the argmax / argmin form (compare, select, select over a value and an iota) is supported";
    if (o.regions.empty() || o.tout.size() != 2) fail(what);
    const auto& region = o.regions[0];
    if (region.empty() || region[0].name != "__block_args__" || region[0].block_args.size() != 4) fail(what);
    const std::string a1 = region[0].block_args[0].first, i1 = region[0].block_args[1].first, a2 = region[0].block_args[2].first,
                      i2 = region[0].block_args[3].first;
    std::vector<const RawOp*> body;
    for (size_t k = 1; k < region.size(); ++k) body.push_back(&region[k]);
    if (body.size() != 4) fail(what);
    auto short_name = [](const RawOp& r) { return r.name.rfind("stablehlo.", 0) == 0 ? r.name.substr(10) : r.name; };
    const RawOp &cmp = *body[0], &s0 = *body[1], &s1 = *body[2], &ret = *body[3];
    if (short_name(cmp) != "compare" || short_name(s0) != "select" || short_name(s1) != "select" || short_name(ret) != "return") fail(what);
    if (cmp.operands.size() != 2 || cmp.operands[0] != a1 || cmp.operands[1] != a2 || cmp.results.size() != 1) fail(what);
    const std::string c = cmp.results[0];
    const RawOp *sv = nullptr, *si = nullptr;
    for (const RawOp* sel : {&s0, &s1}) {
      if (sel->operands.size() != 3 || sel->operands[0] != c || sel->results.size() != 1) fail(what);
      if (sel->operands[1] == a1 && sel->operands[2] == a2) sv = sel;
      else if (sel->operands[1] == i1 && sel->operands[2] == i2) si = sel;
    }
    if (!sv || !si || ret.operands.size() != 2 || ret.operands[0] != sv->results[0] || ret.operands[1] != si->results[0]) fail(what);
    const std::string dir = cmp.sa.count("direction") ? cmp.sa.at("direction") : "";
    const bool is_max = dir == "GE" || dir == "GT", is_min = dir == "LE" || dir == "LT";
    if (!is_max && !is_min) fail(what);
    const bool first = dir == "GE" || dir == "LE";
    const std::vector<int64_t> dims = o.ia.at("dimensions");
    const Node& idx = g.nodes[in[1]];
    if (dims.size() != 1 || idx.k != OpK::Iota || idx.a0.empty() || idx.a0[0] != dims[0]) fail(what);
    const TType xt = ty(in[0]), it = ty(in[1]);
    if (xt.dims != it.dims || !is_int_dt(it.dt) || it.dt == DT::I1 || ty(in[2]).rank() != 0 || ty(in[3]).rank() != 0) fail(what);
    std::vector<int64_t> kept;
    for (int k = 0; k < xt.rank(); ++k) if (k != dims[0]) kept.push_back(xt.dims[k]);
    if (o.tout[0].dims != kept || o.tout[1].dims != kept || o.tout[0].dt != xt.dt || o.tout[1].dt != it.dt) fail("reduce: result type mismatch");
    Node m;
    m.k = OpK::Reduce;
    m.red = is_max ? Red::Max : Red::Min;
    m.in = {in[0], in[2]};
    m.a0 = dims;
    m.ty = o.tout[0];
    const int mv = g.add(m);
    // positions that hold the extreme keep their index, the others the neutral index
    Node mb;
    mb.k = OpK::BroadcastInDim;
    mb.in = {mv};
    mb.ty = xt;
    for (int k = 0; k < xt.rank(); ++k) if (k != dims[0]) mb.a0.push_back(k);
    const int mbv = g.add(mb);
    Node eq;
    eq.k = OpK::Compare;
    eq.op = "EQ";
    eq.in = {in[0], mbv};
    eq.ty = TType{DT::I1, xt.dims};
    const int eqv = g.add(eq);
    Node lim;
    lim.k = OpK::Constant;
    lim.splat = true;
    lim.ty = TType{it.dt, {}};
    lim.data.assign((size_t)info(it.dt).size, 0);
    {
      const int bits = 8 * info(it.dt).size;
      const bool sgn = info(it.dt).is_signed;
      uint64_t v;
      if (first) v = sgn ? ((uint64_t)1 << (bits - 1)) - 1 : (bits == 64 ? ~(uint64_t)0 : ((uint64_t)1 << bits) - 1);
      else v = sgn ? (uint64_t)1 << (bits - 1) : 0;   // smallest value (two's complement bit pattern)
      memcpy(lim.data.data(), &v, (size_t)info(it.dt).size);
    }
    const int limv = g.add(lim);
    Node limb;
    limb.k = OpK::BroadcastInDim;
    limb.in = {limv};
    limb.ty = it;
    const int limbv = g.add(limb);
    Node sel;
    sel.k = OpK::Select;
    sel.in = {eqv, in[1], limbv};
    sel.ty = it;
    const int selv = g.add(sel);
    Node r;
    r.k = OpK::Reduce;
    r.red = first ? Red::Min : Red::Max;
    r.in = {selv, limv};
    r.a0 = dims;
    r.ty = o.tout[1];
    (void)in[3];
    return {mv, g.add(r)};
  }

  struct ConvDims { int d0 = -1, d1 = -1; std::vector<int> sp; };
  // "[b, f, 1, 0]x[o, i, 1, 0]->[b, f, 1, 0]": position of the two named roles and of every spatial dim
  static void parse_conv_dims(const std::string& text, ConvDims out[3]) {
    size_t pos = 0;
    const char* names[3] = {"bf", "oi", "bf"};
    for (int which = 0; which < 3; ++which) {
      size_t b = text.find('[', pos), e = text.find(']', b);
      if (b == std::string::npos || e == std::string::npos) fail("convolution: malformed dimension numbers '" + text + "'");
      std::vector<std::string> toks;
      std::stringstream ss(text.substr(b + 1, e - b - 1));
      std::string tok;
      while (std::getline(ss, tok, ',')) {
        std::string t;
        for (char ch : tok) if (!isspace((unsigned char)ch)) t += ch;
        toks.push_back(t);
      }
      if (toks.size() < 2) fail("convolution: malformed dimension numbers '" + text + "'");
      out[which].sp.assign(toks.size() - 2, -1);
      for (size_t k = 0; k < toks.size(); ++k) {
        if (toks[k].size() == 1 && toks[k][0] == names[which][0]) out[which].d0 = (int)k;
        else if (toks[k].size() == 1 && toks[k][0] == names[which][1]) out[which].d1 = (int)k;
        else {
          int64_t v = -1;
          try { v = std::stoll(toks[k]); } catch (...) { v = -1; }
          if (v < 0 || v >= (int64_t)out[which].sp.size() || out[which].sp[v] >= 0) fail("convolution: malformed dimension numbers '" + text + "'");
          out[which].sp[v] = (int)k;
        }
      }
      if (out[which].d0 < 0 || out[which].d1 < 0) fail("convolution: malformed dimension numbers '" + text + "'");
      for (int v : out[which].sp) if (v < 0) fail("convolution: malformed dimension numbers '" + text + "'");
      pos = e + 1;
    }
  }

  // convolution (reference src/Ops.jl:1000-1073; NNlib's conv, ext/ReactantNNlibExt/Implementations.jl:42-79).
  // It becomes one matrix product on the MFMA path: the weights [O, I*taps] against the matrix of
  // input windows [I*taps, B*outputs] (one batch entry per feature group), which a map kernel writes
  // with coalesced reads along the minor spatial dimension of the input.
  int build_convolution(const RawOp& o_in, int x, int w, const TType& out) {
    RawOp o = o_in;   // window attributes are renumbered below
    if (!o.sa.count("dim_numbers")) fail("convolution: dimension numbers missing");
    ConvDims cd[3];
    parse_conv_dims(o.sa.at("dim_numbers"), cd);
    const TType xt = ty(x), wt = ty(w);
    const int r = xt.rank(), nsp = r - 2;
    if (nsp < 0 || wt.rank() != r || out.rank() != r) fail("convolution: operand ranks do not match");
    for (auto& c : cd) if ((int)c.sp.size() != nsp) fail("convolution: dimension numbers do not match the rank");
    // Number the spatial dims in the order the input stores them, so that the canonical input keeps
    // its minor dimension (reads stay coalesced) and needs no transpose in the usual layouts.
    {
      std::vector<int> order(nsp);
      for (int d = 0; d < nsp; ++d) order[d] = d;
      std::sort(order.begin(), order.end(), [&](int p, int q) { return cd[0].sp[p] < cd[0].sp[q]; });
      auto permute = [&](const char* key) {
        auto itv = o.ia.find(key);
        if (itv == o.ia.end() || (int)itv->second.size() != nsp) return;
        std::vector<int64_t> v(nsp);
        for (int d = 0; d < nsp; ++d) v[d] = itv->second[order[d]];
        o.ia[key] = v;
      };
      for (const char* key : {"window_strides", "lhs_dilation", "rhs_dilation", "window_reversal"}) permute(key);
      auto pv = o.ia.find("padding");
      if (pv != o.ia.end() && (int)pv->second.size() == 2 * nsp) {
        std::vector<int64_t> v(2 * nsp);
        for (int d = 0; d < nsp; ++d) { v[2 * d] = pv->second[2 * order[d]]; v[2 * d + 1] = pv->second[2 * order[d] + 1]; }
        o.ia["padding"] = v;
      }
      for (auto& c : cd) {
        std::vector<int> sp(nsp);
        for (int d = 0; d < nsp; ++d) sp[d] = c.sp[order[d]];
        c.sp = sp;
      }
    }
    if (xt.dt != wt.dt || out.dt != xt.dt) fail("convolution: operand and result element types must match");
    auto get = [&](const char* key, int64_t dflt) {
      std::vector<int64_t> v = o.ia.count(key) ? o.ia.at(key) : std::vector<int64_t>(nsp, dflt);
      if (v.empty()) v.assign(nsp, dflt);
      if ((int)v.size() != nsp) fail(std::string("convolution: ") + key + " must have one entry per spatial dimension");
      return v;
    };
    const auto st = get("window_strides", 1), ld = get("lhs_dilation", 1), rd = get("rhs_dilation", 1), rev = get("window_reversal", 0);
    std::vector<int64_t> pad = o.ia.count("padding") ? o.ia.at("padding") : std::vector<int64_t>(2 * nsp, 0);
    if (pad.size() == 1) pad.assign(2 * nsp, pad[0]);
    if ((int)pad.size() != 2 * nsp) fail("convolution: padding must be a (spatial rank x 2) matrix");
    const int64_t G = o.ia.count("feature_group_count") && !o.ia.at("feature_group_count").empty() ? o.ia.at("feature_group_count")[0] : 1;
    const int64_t BG = o.ia.count("batch_group_count") && !o.ia.at("batch_group_count").empty() ? o.ia.at("batch_group_count")[0] : 1;
    if (BG < 1 || (BG > 1 && G > 1)) fail("convolution: batch_group_count and feature_group_count cannot both exceed 1");
    if (G < 1) fail("convolution: feature_group_count must be positive");

    // canonical orders: input [b, f, s...], kernel [o, i, k...]
    auto canon = [&](int node, const ConvDims& c) {
      std::vector<int64_t> perm{c.d0, c.d1};
      for (int v : c.sp) perm.push_back(v);
      bool identity = true;
      for (size_t k = 0; k < perm.size(); ++k) identity = identity && perm[k] == (int64_t)k;
      if (identity) return node;
      const TType t = ty(node);
      Node n;
      n.k = OpK::Transpose;
      n.in = {node};
      n.a0 = perm;
      n.ty.dt = t.dt;
      for (auto pdim : perm) n.ty.dims.push_back(t.dims[pdim]);
      return g.add(n);
    };
    int xc = canon(x, cd[0]);
    int wc = canon(w, cd[1]);
    {
      std::vector<int64_t> rdims;
      for (int d = 0; d < nsp; ++d) if (rev[d]) rdims.push_back(2 + d);
      if (!rdims.empty()) {
        Node n;
        n.k = OpK::Reverse;
        n.in = {wc};
        n.ty = ty(wc);
        n.a0 = rdims;
        wc = g.add(n);
      }
    }
    const TType xct = ty(xc), wct = ty(wc);
    const int64_t B = xct.dims[0], C = xct.dims[1], O = wct.dims[0], I = wct.dims[1];
    if (C != I * G || O % G != 0) fail("convolution: feature counts do not match feature_group_count");
    if (B % BG != 0 || O % BG != 0) fail("convolution: batch and output feature counts must be multiples of batch_group_count");
    const int64_t Bo = B / BG;    // batch entries of the result
    // f32 images with two spatial dims, no input dilation, no groups and non-negative padding: the direct-convolution
    // kernel (OpK::Conv; rx_conv_body in kernels/rx_gemm_kernels.h) where its tiling covers the shapes
    // 16-bit images with fewer than 16 channels (the first layer of a network: three) take it too, converted to f32 on
    // the way in and back in the kernel's epilogue: their window matrix is all padding, and the products of 16-bit
    // values are exact in f32 (3 -> 64 features, 3 x 3, on 32 x 224^2 bf16: 0.19 ms through the window matrix)
    const bool narrow_stem = (xct.dt == DT::BF16 || xct.dt == DT::F16) && C < 16;
    if (nsp == 2 && (xct.dt == DT::F32 || narrow_stem) && G == 1 && BG == 1 && st[0] >= 1 && st[1] >= 1 && ld[0] == 1 && ld[1] == 1 && rd[0] >= 1 && rd[1] >= 1 &&
        pad[0] >= 0 && pad[1] >= 0 && pad[2] >= 0 && pad[3] >= 0 && wct.dims[2] >= 1 && wct.dims[3] >= 1) {
      const int64_t KH = wct.dims[2], KW = wct.dims[3];
      const int64_t eh = xct.dims[2] + pad[0] + pad[1] - ((KH - 1) * rd[0] + 1), ew = xct.dims[3] + pad[2] + pad[3] - ((KW - 1) * rd[1] + 1);
      const int64_t HO = eh >= 0 ? eh / st[0] + 1 : 0, WO = ew >= 0 ? ew / st[1] + 1 : 0;
      if (HO >= 1 && WO >= 1 && (choose_conv(B, C, xct.dims[2], xct.dims[3], O, KH, KW, HO, WO, pad[2], st[0], st[1], rd[0], rd[1]).ok ||
                                 (split_convs && xct.dt == DT::F32 && conv_split_pays(B, C, xct.dims[2], xct.dims[3], O, KH, KW, HO, WO, pad[2], st[0], st[1], rd[0], rd[1], split_convs == kSplitAlone)))) {
        std::vector<int64_t> want(r);
        want[cd[2].d0] = B; want[cd[2].d1] = O; want[cd[2].sp[0]] = HO; want[cd[2].sp[1]] = WO;
        if (want != out.dims) fail("convolution: result shape mismatch");
        int xf = xc, wf = wc;
        if (narrow_stem) {
          Node c1; c1.k = OpK::Convert; c1.in = {xc}; c1.ty = TType{DT::F32, xct.dims}; xf = g.add(c1);
          Node c2; c2.k = OpK::Convert; c2.in = {wc}; c2.ty = TType{DT::F32, wct.dims}; wf = g.add(c2);
        }
        Node cv;
        cv.k = OpK::Conv;
        cv.in = {xf, wf};
        cv.a0 = {pad[0], pad[1], pad[2], pad[3]};
        cv.a1 = {st[0], st[1]};
        cv.a2 = {rd[0], rd[1]};
        cv.ty = TType{DT::F32, {B, O, HO, WO}};
        int cur = g.add(cv);
        if (narrow_stem) { Node c3; c3.k = OpK::Convert; c3.in = {cur}; c3.ty = TType{out.dt, {B, O, HO, WO}}; cur = g.add(c3); }
        // [B, O, rows, columns] -> the result's own dimension order
        std::vector<int64_t> perm(r);
        perm[cd[2].d0] = 0; perm[cd[2].d1] = 1; perm[cd[2].sp[0]] = 2; perm[cd[2].sp[1]] = 3;
        bool identity = true;
        for (int k = 0; k < r; ++k) identity = identity && perm[k] == k;
        if (!identity) {
          Node t;
          t.k = OpK::Transpose;
          t.in = {cur};
          t.a0 = perm;
          t.ty = out;
          cur = g.add(t);
        }
        if (!(ty(cur) == out)) fail("convolution: internal shape error");
        return cur;
      }
    }
    // 16-bit images with two spatial dims, unit strides, no input dilation, no groups and non-negative padding, whose
    // channels are whole 128-byte K tiles or can be padded to that: the images are zero-padded and laid out [image, row, column, channel], the filter
    // [feature, tap, channel], and the convolution is a matrix product whose first operand is read through one row
    // shift per tap (OpK::Conv with a3; rx_tap_shift in kernels/rx_gemm_kernels.h) -- evaluated on the padded grid,
    // [image, padded row, padded column, feature], from which the result is sliced and transposed.  No window matrix
    // exists.  Taken where the product gets a GEMM skeleton that loads its tiles straight into LDS; RX_CONV_SHIFT=0
    // keeps the window matrix.
    // A strided 1 x 1 filter without padding reads every st-th pixel only: the images are sliced first, and the
    // convolution has unit strides.
    const bool pointwise = nsp == 2 && wct.dims[2] == 1 && wct.dims[3] == 1 && pad[0] == 0 && pad[1] == 0 && pad[2] == 0 && pad[3] == 0 && st[0] >= 1 && st[1] >= 1;
    if (nsp == 2 && (xct.dt == DT::BF16 || xct.dt == DT::F16) && G == 1 && BG == 1 && ((st[0] == 1 && st[1] == 1) || pointwise) && ld[0] == 1 && ld[1] == 1 && rd[0] >= 1 && rd[1] >= 1 &&
        pad[0] >= 0 && pad[1] >= 0 && pad[2] >= 0 && pad[3] >= 0 && wct.dims[2] >= 1 && wct.dims[3] >= 1 && (double)((C + 63) / 64 * 64) <= (getenv("RX_CONV_SHIFT_WASTE") ? atof(getenv("RX_CONV_SHIFT_WASTE")) : 4.0) * (double)C && O % 8 == 0 &&
        !(getenv("RX_CONV_SHIFT") && atoi(getenv("RX_CONV_SHIFT")) == 0) && !(getenv("RX_MFMA") && atoi(getenv("RX_MFMA")) == 0)) {
      const int64_t KH = wct.dims[2], KW = wct.dims[3];
      const int64_t HS = (xct.dims[2] - 1) / st[0] + 1, WS = (xct.dims[3] - 1) / st[1] + 1;   // the images after the slice (unit strides: as they are)
      const int64_t HP = HS + pad[0] + pad[1], WP = WS + pad[2] + pad[3];
      const int64_t HO = HP - (KH - 1) * rd[0], WO = WP - (KW - 1) * rd[1];
      // channels that are not whole K tiles (96, 160; 16, 32) are padded with zero channels to the next multiple of 64, in
      // the images and in the filter, up to four times their number (32 -> 64 features on 32 x 112^2: 0.186 -> 0.099 ms,
      // 16 -> 32 on 16 x 224^2: 0.179 -> 0.121; three channels would be 21 times: 0.19 -> 0.33); RX_CONV_SHIFT_WASTE
      const int64_t CP = (C + 63) / 64 * 64;
      const int64_t MP = B * HP * WP, KK = KH * KW * CP;
      GemmChoice gc;
      // few results and a long contraction: the product on the window matrix is cut along K (split_dots in the planner,
      // the same test), which this form is not (512 -> 512 features on four 14 x 14 images: 0.026 against 0.061 ms)
      const bool sliced = ((B * HO * WO + 63) / 64) * ((O + 63) / 64) < 256 && KK >= 1024 && !(getenv("RX_SPLIT_K") && atoi(getenv("RX_SPLIT_K")) == 0);
      if (HO >= 1 && WO >= 1 && !sliced && MP * CP * 2 < ((int64_t)1 << 31) && O * KK * 2 < ((int64_t)1 << 31) && KH * KW <= 1024)
        gc = choose_gemm(xct.dt, xct.dt, xct.dt, 1, MP, O, KK, true, true, false, 1, false);
      if (gc.ok && (gc.skeleton == "rx_gemm_body_pp" || gc.skeleton == "rx_gemm_body_s" || (gc.skeleton == "rx_gemm_body_dl" && gc.bk * 2 == 128 && gc.split == 1))) {
        std::vector<int64_t> want(r);
        want[cd[2].d0] = B; want[cd[2].d1] = O; want[cd[2].sp[0]] = HO; want[cd[2].sp[1]] = WO;
        if (want != out.dims) fail("convolution: result shape mismatch");
        auto add_node = [&](OpK k, std::vector<int> in, TType t) { Node n; n.k = k; n.in = std::move(in); n.ty = std::move(t); return n; };
        int xi = xc;
        if (st[0] > 1 || st[1] > 1) {
          Node sl = add_node(OpK::Slice, {xi}, TType{xct.dt, {B, C, HS, WS}});
          sl.a0 = {0, 0, 0, 0}; sl.a1 = {B, C, xct.dims[2], xct.dims[3]}; sl.a2 = {1, 1, st[0], st[1]};
          xi = g.add(sl);
        }
        if (pad[0] || pad[1] || pad[2] || pad[3] || CP != C) {
          Node pn = add_node(OpK::Pad, {xi, zero_of(xct.dt)}, TType{xct.dt, {B, CP, HP, WP}});
          pn.a0 = {0, 0, pad[0], pad[2]}; pn.a1 = {0, CP - C, pad[1], pad[3]}; pn.a2 = {0, 0, 0, 0};
          xi = g.add(pn);
        }
        // (the product takes [B, HP, WP, CP] as the matrix [B * HP * WP, CP]: the layout map keeps its four dimensions)
        { Node t = add_node(OpK::Transpose, {xi}, TType{xct.dt, {B, HP, WP, CP}}); t.a0 = {0, 2, 3, 1}; xi = g.add(t); }
        int wi = wc;
        if (CP != C) {
          Node pn = add_node(OpK::Pad, {wi, zero_of(xct.dt)}, TType{xct.dt, {O, CP, KH, KW}});
          pn.a0 = {0, 0, 0, 0}; pn.a1 = {0, CP - C, 0, 0}; pn.a2 = {0, 0, 0, 0};
          wi = g.add(pn);
        }
        { Node t = add_node(OpK::Transpose, {wi}, TType{xct.dt, {O, KH, KW, CP}}); t.a0 = {0, 2, 3, 1}; wi = g.add(t); }
        wi = g.add(add_node(OpK::Reshape, {wi}, TType{xct.dt, {O, KK}}));
        // the kernel's epilogue keeps the rows of the padded grid that are results and writes them side by side:
        // [B, HO, WO, O]
        Node cv = add_node(OpK::Conv, {xi, wi}, TType{out.dt, {B, HO, WO, O}});
        cv.a3 = {KW, rd[0] * WP, rd[1], HP, WP};
        int cur = g.add(cv);
        // [B, rows, columns, O] -> the result's own dimension order
        std::vector<int64_t> perm(r);
        perm[cd[2].d0] = 0; perm[cd[2].d1] = 3; perm[cd[2].sp[0]] = 1; perm[cd[2].sp[1]] = 2;
        bool identity = true;
        for (int k = 0; k < r; ++k) identity = identity && perm[k] == k;
        if (!identity) {
          Node t = add_node(OpK::Transpose, {cur}, out);
          t.a0 = perm;
          cur = g.add(t);
        }
        if (!(ty(cur) == out)) fail("convolution: internal shape error");
        return cur;
      }
    }
    // dilate and pad the input
    {
      std::vector<int64_t> lo(r, 0), hi(r, 0), interior(r, 0);
      bool any = false;
      // negative padding (the gradient forms produce it) crops the dilated input: pad by the
      // non-negative parts, then slice the rest off
      std::vector<int64_t> crop_lo(r, 0), crop_hi(r, 0);
      bool any_crop = false;
      for (int d = 0; d < nsp; ++d) {
        if (ld[d] < 1) fail("convolution: lhs_dilation must be positive");
        lo[2 + d] = std::max<int64_t>(pad[2 * d], 0); hi[2 + d] = std::max<int64_t>(pad[2 * d + 1], 0); interior[2 + d] = ld[d] - 1;
        crop_lo[2 + d] = std::max<int64_t>(-pad[2 * d], 0); crop_hi[2 + d] = std::max<int64_t>(-pad[2 * d + 1], 0);
        any = any || lo[2 + d] || hi[2 + d] || interior[2 + d];
        any_crop = any_crop || crop_lo[2 + d] || crop_hi[2 + d];
      }
      if (any) {
        Node pn;
        pn.k = OpK::Pad;
        pn.in = {xc, zero_of(xct.dt)};
        pn.a0 = lo; pn.a1 = hi; pn.a2 = interior;
        pn.ty.dt = xct.dt;
        for (int d = 0; d < r; ++d) pn.ty.dims.push_back(lo[d] + hi[d] + xct.dims[d] + std::max<int64_t>(xct.dims[d] - 1, 0) * interior[d]);
        xc = g.add(pn);
      }
      if (any_crop) {
        const TType t = ty(xc);
        Node sl;
        sl.k = OpK::Slice;
        sl.in = {xc};
        sl.a0 = crop_lo;
        sl.a2.assign(r, 1);
        sl.ty.dt = t.dt;
        for (int d = 0; d < r; ++d) {
          const int64_t lim = t.dims[d] - crop_hi[d];
          if (lim < crop_lo[d]) fail("convolution: negative padding removes more than the input holds");
          sl.a1.push_back(lim);
          sl.ty.dims.push_back(lim - crop_lo[d]);
        }
        xc = g.add(sl);
      }
    }
    std::vector<int64_t> wsz{1, 1}, wst{1, 1}, wdl{1, 1};
    int64_t taps = 1;
    for (int d = 0; d < nsp; ++d) { wsz.push_back(wct.dims[2 + d]); wst.push_back(st[d]); wdl.push_back(rd[d]); taps *= wct.dims[2 + d]; }
    const int win = window_view(xc, wsz, wst, wdl, "convolution");     // [1, 1, k..., B, C, o...]
    const TType wint = ty(win);
    std::vector<int64_t> osp(wint.dims.begin() + r + 2, wint.dims.end());
    int64_t P = 1;
    for (auto v : osp) P *= v;
    // expected result shape
    {
      std::vector<int64_t> want(r);
      want[cd[2].d0] = Bo; want[cd[2].d1] = O;
      for (int d = 0; d < nsp; ++d) want[cd[2].sp[d]] = osp[d];
      if (want != out.dims) fail("convolution: result shape mismatch");
    }
    if (out.numel() == 0 || taps * I == 0) {
      // nothing to contract or nothing to produce: zeros
      Node bz;
      bz.k = OpK::BroadcastInDim;
      bz.in = {zero_of(out.dt)};
      bz.ty = out;
      return g.add(bz);
    }
    // [k..., B, C, o...] -> [C, k..., B, o...]: rows of the window matrix are (feature, tap), columns (batch entry, output)
    std::vector<int64_t> d1(wint.dims.begin() + 2, wint.dims.end());
    int cur = add_node(OpK::Reshape, TType{xct.dt, d1}, {win});
    {
      Node t;
      t.k = OpK::Transpose;
      t.in = {cur};
      t.a0.push_back(nsp + 1);
      for (int d = 0; d < nsp; ++d) t.a0.push_back(d);
      t.a0.push_back(nsp);
      for (int d = 0; d < nsp; ++d) t.a0.push_back(nsp + 2 + d);
      t.ty.dt = xct.dt;
      for (auto pdim : t.a0) t.ty.dims.push_back(d1[pdim]);
      cur = g.add(t);
    }
    // batch groups (the filter gradient of a grouped convolution): output features of group g see only
    // the batch entries of group g, i.e. one product per group: [C, k..., (g, b'), o...] -> [g, C, k..., b', o...]
    if (BG > 1) {
      const TType t = ty(cur);
      std::vector<int64_t> sd;
      for (int d = 0; d <= nsp; ++d) sd.push_back(t.dims[d]);
      sd.push_back(BG);
      sd.push_back(Bo);
      for (int d = 0; d < nsp; ++d) sd.push_back(t.dims[nsp + 2 + d]);
      cur = add_node(OpK::Reshape, TType{t.dt, sd}, {cur});
      Node tr;
      tr.k = OpK::Transpose;
      tr.in = {cur};
      tr.a0.push_back(nsp + 1);
      for (int d = 0; d <= nsp; ++d) tr.a0.push_back(d);
      for (int d = nsp + 2; d < (int)sd.size(); ++d) tr.a0.push_back(d);
      tr.ty.dt = t.dt;
      for (auto pdim : tr.a0) tr.ty.dims.push_back(sd[pdim]);
      cur = g.add(tr);
    }
    // The MFMA skeletons read 16-byte vectors along the contracted dimension of the weights and along
    // the columns of the window matrix: both are padded with zeros to whole vectors (the extra
    // columns are sliced off the product).
    const int64_t K = I * taps, N = Bo * P;
    int64_t Kp = K, Np = N;
    if (xct.dt == DT::F32 || xct.dt == DT::BF16 || xct.dt == DT::F16 || xct.dt == DT::F64) {
      const int64_t ve = std::max<int64_t>(4, 16 / info(xct.dt).size);
      Kp = (K + ve - 1) / ve * ve;
      Np = (N + ve - 1) / ve * ve;
    }
    auto padded = [&](int node, std::vector<int64_t> hi) {
      bool any = false;
      for (auto v : hi) any = any || v != 0;
      if (!any) return node;
      const TType t = ty(node);
      Node pn;
      pn.k = OpK::Pad;
      pn.in = {node, zero_of(t.dt)};
      pn.a0.assign(t.rank(), 0);
      pn.a1 = hi;
      pn.a2.assign(t.rank(), 0);
      pn.ty.dt = t.dt;
      for (int d = 0; d < t.rank(); ++d) pn.ty.dims.push_back(t.dims[d] + hi[d]);
      return g.add(pn);
    };
    Node dot;
    dot.k = OpK::DotGeneral;
    int lhs, rhs;
    if (BG > 1) {
      lhs = padded(add_node(OpK::Reshape, TType{xct.dt, {BG, O / BG, K}}, {wc}), {0, 0, Kp - K});
      rhs = padded(add_node(OpK::Reshape, TType{xct.dt, {BG, K, N}}, {cur}), {0, Kp - K, Np - N});
      dot.a0 = {0}; dot.a1 = {0}; dot.a2 = {2}; dot.a3 = {1};
      dot.ty = TType{out.dt, {BG, O / BG, Np}};
    } else if (G == 1) {
      lhs = padded(add_node(OpK::Reshape, TType{xct.dt, {O, K}}, {wc}), {0, Kp - K});
      rhs = padded(add_node(OpK::Reshape, TType{xct.dt, {K, N}}, {cur}), {Kp - K, Np - N});
      dot.a2 = {1}; dot.a3 = {0};
      dot.ty = TType{out.dt, {O, Np}};
    } else {
      lhs = padded(add_node(OpK::Reshape, TType{xct.dt, {G, O / G, K}}, {wc}), {0, 0, Kp - K});
      rhs = padded(add_node(OpK::Reshape, TType{xct.dt, {G, K, N}}, {cur}), {0, Kp - K, Np - N});
      dot.a0 = {0}; dot.a1 = {0}; dot.a2 = {2}; dot.a3 = {1};
      dot.ty = TType{out.dt, {G, O / G, Np}};
    }
    dot.in = {lhs, rhs};
    cur = g.add(dot);
    if (Np != N) {
      Node sl;
      sl.k = OpK::Slice;
      sl.in = {cur};
      const TType t = ty(cur);
      sl.a0.assign(t.rank(), 0);
      sl.a1 = t.dims;
      sl.a1.back() = N;
      sl.a2.assign(t.rank(), 1);
      sl.ty = t;
      sl.ty.dims.back() = N;
      cur = g.add(sl);
    }
    // [O, B, o...] -> the result's own dimension order
    std::vector<int64_t> obd{O, Bo};
    for (auto v : osp) obd.push_back(v);
    std::vector<int64_t> perm(r);
    perm[cd[2].d0] = 1; perm[cd[2].d1] = 0;
    for (int d = 0; d < nsp; ++d) perm[cd[2].sp[d]] = 2 + d;
    bool same_order = true;   // dims of more than one element keep their order: a reshape is enough
    {
      int64_t last = -1;
      for (int k = 0; k < r; ++k)
        if (obd[perm[k]] != 1) { same_order = same_order && perm[k] > last; last = perm[k]; }
    }
    if (same_order) {
      cur = add_node(OpK::Reshape, out, {cur});
    } else {
      cur = add_node(OpK::Reshape, TType{out.dt, obd}, {cur});
      Node t;
      t.k = OpK::Transpose;
      t.in = {cur};
      t.a0 = perm;
      t.ty = out;
      cur = g.add(t);
    }
    if (!(ty(cur) == out)) fail("convolution: internal shape error");
    return cur;
  }

  // custom_call of one of the library's own operators (rx_lm.h)
  std::vector<int> build_operator(const RawOp& o, const std::vector<int>& in) {
    OperatorSpec spec;
    spec.name = o.sa.count("call_target_name") ? o.sa.at("call_target_name") : "";
    if (spec.name.size() >= 2 && spec.name.front() == '"' && spec.name.back() == '"') spec.name = spec.name.substr(1, spec.name.size() - 2);
    if (!is_operator_name(spec.name)) fail("custom_call: unknown target '" + spec.name + "'");
    if (o.sa.count("backend_config")) {
      std::string body = o.sa.at("backend_config");
      if (!body.empty() && body.front() == '{') {
        body = body.substr(1, body.size() - 2);
        Cur a(body.c_str(), body.size());
        while (!a.eof()) {
          const std::string key = a.ident();
          a.expect("=");
          const std::string v = a.value();
          if (a.accept(":")) a.value();
          if (!spec.attrs.emplace(key, v).second) fail(spec.name + ": setting '" + key + "' is given twice");
          if (!a.accept(",") && !a.eof()) a.fail("expected ','");
        }
      } else if (!body.empty()) {
        fail(spec.name + ": backend_config must be a dictionary");
      }
    }
    for (int i : in) spec.in.push_back(ty(i));
    spec.out = o.tout;
    if (o.tin.size() != in.size()) fail(spec.name + ": one type per operand expected");
    for (size_t k = 0; k < in.size(); ++k)
      if (!(o.tin[k] == spec.in[k])) fail(spec.name + ": operand " + std::to_string(k) + " has type " + spec.in[k].str() + ", declared " + o.tin[k].str());
    check_operator(spec);
    Node n;
    n.k = OpK::Operator;
    n.op = spec.name;
    n.attrs = spec.attrs;
    n.in = in;
    n.ty = spec.out[0];
    n.a0 = {(int64_t)spec.out.size()};
    std::vector<int> res{g.add(n)};
    for (size_t r = 1; r < spec.out.size(); ++r) {
      const int id = add_node(OpK::OperatorResult, spec.out[r], {res[0]});
      g.nodes[id].a0 = {(int64_t)r};
      res.push_back(id);
    }
    return res;
  }

  std::vector<int> build(const RawOp& o, const std::vector<int>& in, int depth) {
    std::string sh = o.name;
    if (sh.rfind("stablehlo.", 0) == 0) sh = sh.substr(10);
    auto need = [&](size_t k) { if (in.size() != k) fail(o.name + ": expected " + std::to_string(k) + " operands"); };
    auto out1 = [&]() -> const TType& { if (o.tout.size() != 1) fail(o.name + ": expected one result type"); return o.tout[0]; };
    Node n;
    n.in = in;
    if (sh == "optimization_barrier") return in;
    if (sh == "custom_call") return build_operator(o, in);
    if (sh == "call") {
      auto it = p.funcs.find(o.sa.at("callee"));
      if (it == p.funcs.end()) fail("call to unknown function @" + o.sa.at("callee"));
      return inline_func(it->second, in, depth + 1);
    }
    if (sh == "constant") {
      n.k = OpK::Constant;
      n.ty = out1();
      fill_constant(n, o.dense, [&](const std::string& m) { fail("constant: " + m); });
      return {g.add(n)};
    }
    if (in_list(kUnary, sh) || in_list(kChloUnary, sh)) {
      need(1);
      n.k = OpK::Unary;
      n.op = sh.rfind("chlo.", 0) == 0 ? sh.substr(5) : sh;
      n.ty = out1();
      if (sh == "is_finite" || sh == "chlo.is_inf" || sh == "chlo.is_pos_inf" || sh == "chlo.is_neg_inf") n.ty.dt = DT::I1;
      if (in_list(kChloUnary, sh) && !is_float(ty(in[0]).dt)) fail(o.name + ": a float operand is expected");
      if (n.ty.dims != ty(in[0]).dims) fail(o.name + ": shape mismatch");
      return {g.add(n)};
    }
    if (sh == "enzymexla.math.gelu") {
      need(1);
      n.k = OpK::Gelu;
      n.op = o.sa.count("approximation") ? o.sa.at("approximation") : (o.sa.count("gelu_approximation") ? o.sa.at("gelu_approximation") : "NONE");
      n.ty = out1();
      check_same(n.ty, ty(in[0]), o.name);
      return {g.add(n)};
    }
    if (in_list(kBinary, sh)) {
      need(2);
      n.k = OpK::Binary;
      n.op = sh;
      n.ty = out1();
      check_same(ty(in[0]), ty(in[1]), o.name);
      check_same(n.ty, ty(in[0]), o.name);
      return {g.add(n)};
    }
    if (sh == "bitcast_convert") {
      // the same bits as another type of the same width (32- and 64-bit types, 8/16-bit integers)
      need(1);
      n.k = OpK::Unary;
      n.op = "bitcast";
      n.ty = out1();
      const DT s_ = ty(in[0]).dt, d_ = n.ty.dt;
      if (n.ty.dims != ty(in[0]).dims || info(s_).size != info(d_).size || is_narrow_float(s_) || is_narrow_float(d_) || s_ == DT::I1 || d_ == DT::I1)
        fail("bitcast_convert: only between types of one width (no 8/16-bit floats, no i1)");
      return {g.add(n)};
    }
    if (sh == "get_dimension_size") {
      need(1);
      if (!o.ia.count("dimension") || o.ia.at("dimension").empty()) fail("get_dimension_size: dimension missing");
      const int64_t d_ = o.ia.at("dimension")[0];
      if (d_ < 0 || d_ >= ty(in[0]).rank()) fail("get_dimension_size: dimension out of range");
      return {splat_of(out1(), (double)ty(in[0]).dims[d_])};
    }
    if (sh == "convert") {
      need(1);
      n.k = OpK::Convert;
      n.ty = out1();
      if (n.ty.dims != ty(in[0]).dims) fail("convert: shape mismatch");
      return {g.add(n)};
    }
    if (sh == "compare") {
      need(2);
      n.k = OpK::Compare;
      n.op = o.sa.at("direction");
      n.ty = ty(in[0]);
      n.ty.dt = DT::I1;
      check_same(ty(in[0]), ty(in[1]), "compare");
      return {g.add(n)};
    }
    if (sh == "select") {
      need(3);
      n.k = OpK::Select;
      n.ty = ty(in[1]);
      check_same(ty(in[1]), ty(in[2]), "select");
      if (ty(in[0]).dt != DT::I1) fail("select: predicate must be i1");
      if (ty(in[0]).rank() != 0 && ty(in[0]).dims != n.ty.dims) fail("select: predicate shape mismatch");
      return {g.add(n)};
    }
    if (sh == "clamp") {
      need(3);
      n.k = OpK::Clamp;
      n.ty = ty(in[1]);
      for (int k : {0, 2})
        if (ty(in[k]).rank() != 0 && ty(in[k]).dims != n.ty.dims) fail("clamp: bound shape mismatch");
      return {g.add(n)};
    }
    if (sh == "broadcast_in_dim") {
      need(1);
      n.k = OpK::BroadcastInDim;
      n.ty = out1();
      n.a0 = o.ia.count("broadcast_dimensions") ? o.ia.at("broadcast_dimensions") : std::vector<int64_t>{};
      const TType& s = ty(in[0]);
      if ((int)n.a0.size() != s.rank()) fail("broadcast_in_dim: dims/operand rank mismatch");
      for (int k = 0; k < s.rank(); ++k) {
        int64_t d = n.a0[k];
        if (d < 0 || d >= n.ty.rank()) fail("broadcast_in_dim: dimension out of range");
        if (s.dims[k] != 1 && s.dims[k] != n.ty.dims[d]) fail("broadcast_in_dim: size mismatch");
      }
      if (s.dt != n.ty.dt) fail("broadcast_in_dim: element type mismatch");
      return {g.add(n)};
    }
    if (sh == "reshape") {
      need(1);
      n.k = OpK::Reshape;
      n.ty = out1();
      if (n.ty.numel() != ty(in[0]).numel()) fail("reshape: element count mismatch");
      return {g.add(n)};
    }
    if (sh == "transpose") {
      need(1);
      n.k = OpK::Transpose;
      n.ty = out1();
      n.a0 = o.ia.at("permutation");
      const TType& s = ty(in[0]);
      if ((int)n.a0.size() != s.rank() || n.ty.rank() != s.rank()) fail("transpose: rank mismatch");
      for (int k = 0; k < s.rank(); ++k)
        if (n.a0[k] < 0 || n.a0[k] >= s.rank() || n.ty.dims[k] != s.dims[n.a0[k]]) fail("transpose: bad permutation");
      return {g.add(n)};
    }
    if (sh == "slice") {
      need(1);
      n.k = OpK::Slice;
      n.ty = out1();
      n.a0 = o.ia.at("start_indices");
      n.a1 = o.ia.at("limit_indices");
      n.a2 = o.ia.count("strides") ? o.ia.at("strides") : std::vector<int64_t>(n.a0.size(), 1);
      const TType& s = ty(in[0]);
      if ((int)n.a0.size() != s.rank()) fail("slice: rank mismatch");
      for (int k = 0; k < s.rank(); ++k) {
        if (n.a0[k] < 0 || n.a1[k] > s.dims[k] || n.a0[k] > n.a1[k] || n.a2[k] < 1) fail("slice: bounds out of range");
        int64_t sz = (n.a1[k] - n.a0[k] + n.a2[k] - 1) / n.a2[k];
        if (sz != n.ty.dims[k]) fail("slice: result shape mismatch");
      }
      return {g.add(n)};
    }
    if (sh == "pad") {
      need(2);
      n.k = OpK::Pad;
      n.ty = out1();
      n.a0 = o.ia.at("edge_padding_low");
      n.a1 = o.ia.at("edge_padding_high");
      n.a2 = o.ia.at("interior_padding");
      const TType& s = ty(in[0]);
      if (ty(in[1]).rank() != 0) fail("pad: padding value must be 0-d");
      for (int k = 0; k < s.rank(); ++k) {
        if (n.a2[k] < 0) fail("pad: negative interior padding");
        int64_t span = s.dims[k] + std::max<int64_t>(s.dims[k] - 1, 0) * n.a2[k];
        if (n.a0[k] + span + n.a1[k] != n.ty.dims[k]) fail("pad: result shape mismatch");
      }
      return {g.add(n)};
    }
    if (sh == "dynamic_update_slice") {
      n.k = OpK::DynamicUpdateSlice;
      n.ty = ty(in[0]);
      if ((int)in.size() != 2 + n.ty.rank()) fail("dynamic_update_slice: index count mismatch");
      for (int k = 0; k < n.ty.rank(); ++k)
        if (ty(in[1]).dims[k] > n.ty.dims[k]) fail("dynamic_update_slice: update larger than operand");
      return {g.add(n)};
    }
    if (sh == "dynamic_slice") {
      n.k = OpK::DynamicSlice;
      n.ty = out1();
      n.a0 = o.ia.at("slice_sizes");
      if ((int)in.size() != 1 + ty(in[0]).rank()) fail("dynamic_slice: index count mismatch");
      return {g.add(n)};
    }
    if (sh == "concatenate") {
      n.k = OpK::Concatenate;
      n.ty = out1();
      n.a0 = o.ia.at("dimension");
      int64_t tot = 0;
      for (int id : in) tot += ty(id).dims[n.a0[0]];
      if (tot != n.ty.dims[n.a0[0]]) fail("concatenate: result shape mismatch");
      return {g.add(n)};
    }
    if (sh == "iota") {
      n.k = OpK::Iota;
      n.ty = out1();
      n.a0 = o.ia.count("iota_dimension") ? o.ia.at("iota_dimension") : o.ia.at("dimension");
      return {g.add(n)};
    }
    if (sh == "reduce" && in.size() == 4) return build_arg_reduce(o, in);
    if (sh == "reduce") {
      if (in.size() != 2) fail("reduce over more than two operands is not supported");
      n.k = OpK::Reduce;
      n.ty = out1();
      n.a0 = o.ia.at("dimensions");
      n.red = body_kind(o);
      const TType& s = ty(in[0]);
      std::vector<int64_t> kept;
      for (int k = 0; k < s.rank(); ++k)
        if (std::find(n.a0.begin(), n.a0.end(), k) == n.a0.end()) kept.push_back(s.dims[k]);
      if (kept != n.ty.dims) fail("reduce: result shape mismatch");
      if (ty(in[1]).rank() != 0) fail("reduce: init must be 0-d");
      return {g.add(n)};
    }
    if (sh == "reverse") {
      need(1);
      n.k = OpK::Reverse;
      n.ty = out1();
      check_same(n.ty, ty(in[0]), o.name);
      n.a0 = o.ia.at("dimensions");
      for (auto d : n.a0) if (d < 0 || d >= n.ty.rank()) fail("reverse: dimension out of range");
      return {g.add(n)};
    }
    if (sh == "scatter") {
      // one operand / one update tensor; the update computation is an assignment (returns its second
      // argument) or a single monoid op of both arguments (reference src/Ops.jl:2150-2268)
      if (in.size() != 3) fail("scatter over several operands is not supported");
      n.k = OpK::Scatter;
      n.ty = out1();
      const TType &ot = ty(in[0]), &st = ty(in[1]), &ut = ty(in[2]);
      if (!(n.ty == ot) || ut.dt != ot.dt) fail("scatter: operand, updates and result types must agree");
      if (!is_int_dt(st.dt) || st.dt == DT::I1) fail("scatter: indices must be integers");
      auto get = [&](const char* key) { return o.ia.count(key) ? o.ia.at(key) : std::vector<int64_t>{}; };
      n.a0 = get("update_window_dims");
      n.a1 = get("inserted_window_dims");
      n.a2 = get("scatter_dims_to_operand_dims");
      n.a4 = get("index_vector_dim");
      n.a5 = get("input_batching_dims");
      n.a6 = get("scatter_indices_batching_dims");
      if (n.a4.size() != 1) fail("scatter: index_vector_dim missing");
      const int r = ot.rank(), rs = st.rank(), ru = ut.rank(), ivd = (int)n.a4[0];
      if (ivd < 0 || ivd > rs) fail("scatter: index_vector_dim out of range");
      if ((int64_t)n.a2.size() != (ivd < rs ? st.dims[ivd] : 1)) fail("scatter: scatter_dims_to_operand_dims does not match the index vector length");
      if (n.a5.size() != n.a6.size()) fail("scatter: batching dimension lists differ in length");
      auto in_range = [&](const std::vector<int64_t>& v, int hi) { for (auto x : v) if (x < 0 || x >= hi) return false; return true; };
      if (!in_range(n.a0, ru) || !in_range(n.a1, r) || !in_range(n.a2, r) || !in_range(n.a5, r) || !in_range(n.a6, rs)) fail("scatter: dimension number out of range");
      if ((int)(n.a0.size() + n.a1.size() + n.a5.size()) != r) fail("scatter: window dims do not cover the operand");
      // updates shape: scatter dims follow the index tensor (without the index vector), window dims fit the operand
      {
        std::vector<int64_t> sdims;
        for (int q = 0; q < rs; ++q) if (q != ivd) sdims.push_back(st.dims[q]);
        if ((int)(sdims.size() + n.a0.size()) != ru) fail("scatter: updates rank mismatch");
        size_t si = 0, wi = 0;
        std::vector<int> wdim;   // operand dim of each window dim
        for (int d = 0; d < r; ++d)
          if (std::find(n.a1.begin(), n.a1.end(), (int64_t)d) == n.a1.end() && std::find(n.a5.begin(), n.a5.end(), (int64_t)d) == n.a5.end()) wdim.push_back(d);
        for (int d = 0; d < ru; ++d) {
          const bool is_win = std::find(n.a0.begin(), n.a0.end(), (int64_t)d) != n.a0.end();
          if (is_win) { if (ut.dims[d] > ot.dims[wdim[wi++]]) fail("scatter: update window exceeds the operand"); }
          else if (ut.dims[d] != sdims[si++]) fail("scatter: updates shape does not match the indices");
        }
      }
      // update computation
      if (o.regions.empty() || o.regions[0].empty() || o.regions[0][0].name != "__block_args__" || o.regions[0][0].block_args.size() != 2)
        fail("scatter: update computation with two arguments expected");
      const auto& region = o.regions[0];
      const std::string a_cur = region[0].block_args[0].first, a_upd = region[0].block_args[1].first;
      std::vector<const RawOp*> body;
      for (size_t k = 1; k < region.size(); ++k) body.push_back(&region[k]);
      if (body.size() == 1 && body[0]->operands.size() == 1 && body[0]->operands[0] == a_upd) n.op = "assign";
      else if (body.size() == 2 && body[0]->operands.size() == 2 && body[1]->operands.size() == 1 && body[0]->results.size() == 1 &&
               body[1]->operands[0] == body[0]->results[0] &&
               ((body[0]->operands[0] == a_cur && body[0]->operands[1] == a_upd) || (body[0]->operands[0] == a_upd && body[0]->operands[1] == a_cur))) {
        const std::string bname = body[0]->name.substr(body[0]->name.rfind('.') + 1);
        const bool in_order = body[0]->operands[0] == a_cur;
        // element - update and element / update (NNlib.scatter!(-, ...) and (/, ...), reference
        // ext/ReactantNNlibExt/Implementations.jl:477-530): the order of the updates of one element
        // does not matter to the exact result, as for the monoids
        if (bname == "subtract" && in_order && ot.dt != DT::I1) n.op = "subtract";
        else if (bname == "divide" && in_order && is_float(ot.dt)) n.op = "divide";
        else {
          RawOp tmp;
          tmp.sa["body"] = bname;
          n.red = body_kind(tmp);
          n.op = "combine";
        }
      } else fail("scatter: the update computation must return its second argument or one op of both (a monoid, element - update, element / update)");
      if (n.op != "assign" && is_narrow_float(ot.dt)) fail("scatter: combining updates of 8- or 16-bit floats is not supported");
      return {g.add(n)};
    }
    if (sh == "gather") {
      need(2);
      n.k = OpK::Gather;
      n.ty = out1();
      const TType& ot = ty(in[0]);
      const TType& st = ty(in[1]);
      auto get = [&](const char* key) { return o.ia.count(key) ? o.ia.at(key) : std::vector<int64_t>{}; };
      n.a0 = get("offset_dims");
      n.a1 = get("collapsed_slice_dims");
      n.a2 = get("start_index_map");
      n.a3 = get("slice_sizes");
      n.a4 = get("index_vector_dim");
      n.a5 = get("operand_batching_dims");
      n.a6 = get("start_indices_batching_dims");
      if (n.a4.size() != 1) fail("gather: index_vector_dim missing");
      const int r = ot.rank(), rs = st.rank(), ivd = (int)n.a4[0];
      if (!is_int_dt(st.dt) || st.dt == DT::I1) fail("gather: start indices must be integers");
      if ((int)n.a3.size() != r) fail("gather: slice_sizes must have one entry per operand dimension");
      if (ivd < 0 || ivd > rs) fail("gather: index_vector_dim out of range");
      if ((int64_t)n.a2.size() != (ivd < rs ? st.dims[ivd] : 1)) fail("gather: start_index_map does not match the index vector length");
      if (n.a5.size() != n.a6.size()) fail("gather: batching dimension lists differ in length");
      auto in_range = [&](const std::vector<int64_t>& v, int hi) { for (auto x : v) if (x < 0 || x >= hi) return false; return true; };
      if (!in_range(n.a1, r) || !in_range(n.a2, r) || !in_range(n.a5, r) || !in_range(n.a6, rs) || !in_range(n.a0, n.ty.rank())) fail("gather: dimension number out of range");
      for (int d = 0; d < r; ++d) {
        if (n.a3[d] < 0 || n.a3[d] > ot.dims[d]) fail("gather: slice size exceeds the operand");
        const bool dropped = std::find(n.a1.begin(), n.a1.end(), (int64_t)d) != n.a1.end() || std::find(n.a5.begin(), n.a5.end(), (int64_t)d) != n.a5.end();
        if (dropped && n.a3[d] != 1) fail("gather: collapsed and batching dimensions need slice size 1");
      }
      // result shape: batch dims of the start indices (without the index vector) interleaved with the kept slice sizes
      {
        std::vector<int64_t> bdims, odims;
        for (int q = 0; q < rs; ++q) if (q != ivd) bdims.push_back(st.dims[q]);
        for (int d = 0; d < r; ++d) {
          const bool dropped = std::find(n.a1.begin(), n.a1.end(), (int64_t)d) != n.a1.end() || std::find(n.a5.begin(), n.a5.end(), (int64_t)d) != n.a5.end();
          if (!dropped) odims.push_back(n.a3[d]);
        }
        if (n.a0.size() != odims.size() || (int)(bdims.size() + odims.size()) != n.ty.rank()) fail("gather: result rank mismatch");
        size_t bi = 0, oi2 = 0;
        for (int d = 0; d < n.ty.rank(); ++d) {
          const bool is_off = std::find(n.a0.begin(), n.a0.end(), (int64_t)d) != n.a0.end();
          const int64_t want = is_off ? odims[oi2++] : bdims[bi++];
          if (n.ty.dims[d] != want) fail("gather: result shape mismatch");
        }
      }
      if (n.ty.dt != ot.dt) fail("gather: element type mismatch");
      return {g.add(n)};
    }
    if (sh == "batch_norm_inference" || sh == "batch_norm_training") return build_batch_norm(o, in, sh == "batch_norm_training");
    if (sh == "reduce_window") {
      if (in.size() != 2) fail("variadic reduce_window is not supported");
      return {build_reduce_window(o, in[0], in[1], out1())};
    }
    if (sh == "select_and_scatter") {
      need(3);
      return {build_select_and_scatter(o, in[0], in[1], in[2], out1())};
    }
    if (sh == "convolution") {
      need(2);
      return {build_convolution(o, in[0], in[1], out1())};
    }
    if (sh == "map") {
      // elementwise application of a scalar body: inline the body on full tensors
      if (o.regions.empty() || o.regions[0].empty()) fail("map without a body");
      auto& region = o.regions[0];
      std::map<std::string, int> env;
      auto& ba = region[0].block_args;
      if (ba.size() != in.size()) fail("map: body argument count mismatch");
      for (size_t k = 0; k < in.size(); ++k) env[ba[k].first] = in[k];
      std::vector<RawOp> body;
      const TType& full = ty(in[0]);
      for (size_t k = 1; k < region.size(); ++k) {
        RawOp r = region[k];
        for (auto& t : r.tout) t.dims = full.dims;
        for (auto& t : r.tin) t.dims = full.dims;
        body.push_back(r);
      }
      return run_block(body, env, depth);
    }
    if (sh == "dot_general") {
      need(2);
      n.k = OpK::DotGeneral;
      n.ty = out1();
      n.a0 = o.ia.at("lhs_batching_dimensions");
      n.a1 = o.ia.at("rhs_batching_dimensions");
      n.a2 = o.ia.at("lhs_contracting_dimensions");
      n.a3 = o.ia.at("rhs_contracting_dimensions");
      const TType &l = ty(in[0]), &r = ty(in[1]);
      if (n.a0.size() != n.a1.size() || n.a2.size() != n.a3.size()) fail("dot_general: dimension list mismatch");
      std::vector<int64_t> shape;
      for (size_t k = 0; k < n.a0.size(); ++k) {
        if (l.dims.at(n.a0[k]) != r.dims.at(n.a1[k])) fail("dot_general: batch size mismatch");
        shape.push_back(l.dims[n.a0[k]]);
      }
      for (size_t k = 0; k < n.a2.size(); ++k)
        if (l.dims.at(n.a2[k]) != r.dims.at(n.a3[k])) fail("dot_general: contracting size mismatch");
      auto isin = [](const std::vector<int64_t>& v, int64_t x) { return std::find(v.begin(), v.end(), x) != v.end(); };
      for (int k = 0; k < l.rank(); ++k) if (!isin(n.a0, k) && !isin(n.a2, k)) shape.push_back(l.dims[k]);
      for (int k = 0; k < r.rank(); ++k) if (!isin(n.a1, k) && !isin(n.a3, k)) shape.push_back(r.dims[k]);
      if (shape != n.ty.dims) fail("dot_general: result shape mismatch");
      return {g.add(n)};
    }
    fail("unsupported operation '" + o.name + "'");
  }
};

}  // namespace

Graph parse_module(const char* text, size_t len, SplitConvs split_convs) {
  P p(text, len);
  p.parse();
  const RawFunc* mainf = nullptr;
  auto it = p.funcs.find("main");
  if (it != p.funcs.end()) mainf = &it->second;
  else if (p.func_order.size() == 1) mainf = &p.funcs[p.func_order[0]];
  if (!mainf) throw Error("StableHLO import: module has no @main function");
  Builder b(p);
  b.split_convs = split_convs;
  b.g.name = mainf->name;
  b.g.module_name = p.module_name;
  std::vector<int> args;
  for (size_t k = 0; k < mainf->args.size(); ++k) {
    Node n;
    n.k = OpK::Param;
    n.ty = mainf->args[k].second;
    n.a0 = {(int64_t)k};
    int id = b.g.add(n);
    args.push_back(id);
    b.g.params.push_back(id);
    int alias = -1;
    const std::string& at = mainf->arg_attrs[k];
    size_t pos = at.find("tf.aliasing_output");
    if (pos != std::string::npos) {
      size_t eq = at.find('=', pos);
      if (eq != std::string::npos) alias = std::stoi(at.substr(eq + 1));
    }
    b.g.aliasing_output.push_back(alias);
  }
  b.g.results = b.inline_func(*mainf, args, 0);
  b.fold_scalar_constants();
  b.keep_loop_slice_starts_in_memory();
  if (b.g.results.size() != mainf->result_types.size()) throw Error("StableHLO import: @main returns the wrong number of values");
  for (size_t k = 0; k < b.g.results.size(); ++k)
    if (!(b.g.nodes[b.g.results[k]].ty == mainf->result_types[k]))
      throw Error("StableHLO import: @main result " + std::to_string(k) + " has type " + b.g.nodes[b.g.results[k]].ty.str() +
                  ", declared " + mainf->result_types[k].str());
  return std::move(b.g);
}

}  // namespace rx
