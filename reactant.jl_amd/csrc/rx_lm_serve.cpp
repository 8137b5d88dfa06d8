// Checks and launches of the norms, of caches that may hold 8 bits, and of the attention of drafted tokens (rx_lm.h).
#include "rx_lm_plan.h"

namespace rx {
namespace lm {
namespace {

constexpr int64_t kMaxNorm = 32768;   // elements of a row: 32 to a lane of the largest workgroup, which stay in registers
constexpr int64_t kMaxSteps = 64;     // of a branch: that many units of four bytes in a thread's registers

bool bits8(DT t) { return t == DT::F8E4M3FN || t == DT::I8; }
const char* stored(DT t) { return t == DT::F8E4M3FN ? "rx_lm_f8" : t == DT::I8 ? "rx_lm_i8" : elem(t); }
std::string cell(const TType& t) { return bits8(t.dt) ? std::string("rx_u8") : st(t); }

void check_eps(const Checker& c) {
  const double v = c.number("eps", 1e-6);
  c.require(v >= 0 && v <= 3.4028234e38, "setting 'eps' must be a number that f32 holds, and not negative");
}

// lanes of a row, elements to a vector, vectors to a lane: at most 16 elements to a lane of a wavefront, 32 of a workgroup
struct Lanes { int64_t lanes, vec, each; };
Lanes lanes_of(int64_t D, int64_t size) {
  Lanes l;
  l.vec = D % (16 / size) == 0 ? 16 / size : 1;
  l.lanes = D <= 1024 ? 64 : D <= 8192 ? 256 : 1024;
  l.each = (D / l.vec + l.lanes - 1) / l.lanes;
  return l;
}

// Caches, their scales (operands k + 2 and k + 3) and the page table, whose caches are operands k and k + 1
void check_stored(const Checker& c, int k, int pages, bool by_slot, DT dt) {
  const auto& in = c.s.in;
  const TType &kt = in[k], &vt = in[k + 1];
  c.rank(kt, 4, "k_cache");
  c.rank(vt, 4, "v_cache");
  c.require(dt == DT::INVALID ? kt.dt == DT::F32 || kt.dt == DT::BF16 || kt.dt == DT::F16 || bits8(kt.dt) : kt.dt == dt || bits8(kt.dt),
            dt == DT::INVALID ? "the caches must be f32, bf16, f16, f8E4M3FN or i8, got " + kt.str() : "the caches must have the type of q, or be f8E4M3FN or i8, got " + kt.str());
  c.require(vt.dt == kt.dt, "the caches must have one type");
  const Cache kc(kt, by_slot), vc(vt, by_slot);
  c.require(kc.pages == vc.pages && kc.slots == vc.slots && kc.heads == vc.heads, "the caches must have the same pages, slots and heads: " + kt.str() + " and " + vt.str());
  c.require(kc.dim >= 1 && kc.dim <= kMaxHeadDim && vc.dim >= 1 && vc.dim <= kMaxHeadDim, "head dimensions from 1 to " + num(kMaxHeadDim) + " are supported");
  c.require(kc.slots >= 1 && kc.slots <= kMaxRow && kc.heads >= 1 && kc.heads <= (1 << 20), "a cache's pages must have slots and heads");
  c.require(kc.pages <= kMaxRow, "the cache has too many pages");
  c.rank(in[pages], 2, "the page table");
  c.ints(in[pages], "the page table");
  c.require(in[pages].dims[1] <= kMaxRow && in[pages].dims[1] * kc.slots <= kMaxRow, "the page table's positions are too many");
  const bool scales = (int)in.size() == k + 4;
  c.require((int)in.size() == k + 2 || scales, "k_scale and v_scale belong together");
  c.require(scales == bits8(kt.dt), scales ? "scales belong to caches of 8 bits" : "caches of 8 bits need k_scale and v_scale");
  for (int i = k + 2; i < (int)in.size(); ++i) {
    c.f32(in[i], i == k + 2 ? "k_scale" : "v_scale");
    c.dims(in[i], {kc.pages, kc.heads, kc.slots}, i == k + 2 ? "k_scale" : "v_scale");
  }
}
bool by_slots(const Checker& c) { return c.word("layout", "slots", {"slots", "heads"}) == "slots"; }

// pairs of each axis
std::vector<int64_t> sections_of(const Checker& c, int64_t axes, int64_t pairs) {
  auto it = c.s.attrs.find("sections");
  std::vector<int64_t> out;
  if (it == c.s.attrs.end()) {
    c.require(axes == 1, "angles of " + num(axes) + " axes need the setting 'sections'");
    return {pairs};
  }
  int64_t sum = 0;
  const char* p = it->second.c_str();
  while (*p) {
    char* end = nullptr;
    const long long v = std::strtoll(p, &end, 10);
    c.require(end != p && *p >= '0' && *p <= '9' && v <= kMaxHeadDim && (*end == 0 || (*end == ',' && end[1])), "setting 'sections' must be whole numbers with commas between them, got '" + it->second + "'");
    out.push_back(v);
    sum += v;
    p = *end ? end + 1 : end;
  }
  c.require((int64_t)out.size() == axes, "setting 'sections' must name one number for each of the " + num(axes) + " axes, got '" + it->second + "'");
  c.require(sum == pairs, "setting 'sections' must add up to the " + num(pairs) + " rotated pairs, got '" + it->second + "'");
  return out;
}

}  // namespace

// ------------------------------------------------------------------ norms
void check_norm(const Checker& c) {
  const auto &in = c.s.in, &out = c.s.out;
  c.settings({"eps"});
  check_eps(c);
  const bool residual = in.size() == 3;
  const TType &x = in[0], &w = in.back();
  c.floats(x, "x");
  c.require(x.rank() >= 1 && x.dims.back() >= 1 && x.dims.back() <= kMaxNorm, "rows of 1 to " + num(kMaxNorm) + " elements are supported, got " + x.str());
  if (residual) c.same(in[0], in[1], "x and residual");
  c.dims(w, {x.dims.back()}, "the weight");
  c.require(w.dt == x.dt, "the weight must have the type of x");
  const size_t at = residual ? 1 : 0;
  c.require(out.size() > at, "wrong number of results: " + num((int64_t)out.size()));
  if (residual) c.same(in[0], out[0], "x and h");
  c.dims(out[at], x.dims, "y");
  c.require(out[at].dt == x.dt || bits8(out[at].dt), "y must have the type of x, or be f8E4M3FN or i8");
  c.require(out.size() == at + (bits8(out[at].dt) ? 2 : 1), bits8(out[at].dt) ? "y of 8 bits needs one result more, its scales" : "scales belong to y of 8 bits");
  if (bits8(out[at].dt)) {
    c.f32(out[at + 1], "the scales");
    c.dims(out[at + 1], without_last(x), "the scales");
  }
  c.require(x.numel() / x.dims.back() <= kMaxRow, "too many rows");
}
OperatorPlan plan_norm(const OperatorSpec& s) {
  const Checker c{s};
  const bool residual = s.in.size() == 3;
  const TType& y = s.out[residual ? 1 : 0];
  const int64_t D = y.dims.back(), rows = y.numel() / D;
  const Lanes l = lanes_of(D, info(s.in[0].dt).size);
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (size_t i = 0; i < s.in.size(); ++i) args.push_back({operand((int)i), st(s.in[i])});
  for (size_t r = 0; r < s.out.size(); ++r) args.push_back({result((int)r), &s.out[r] == &y ? cell(y) : st(s.out[r])});
  const std::string none = "(" + st(s.in[0]) + "*)0", a = residual ? "a0, a1, a2, a3, a4" : "a0, " + none + ", a1, " + none + ", a2";
  OperatorPlan p;
  p.header = "rx_lm_norm_kernels.h";
  OperatorKernel k = kernel(s, "rms_norm", (unsigned)std::max<int64_t>(256, l.lanes), args, (int)s.out.size(),
                            std::string("rx_rms_norm<") + elem(s.in[0].dt) + ", " + stored(y.dt) + ", " + num(D) + ", " + num(rows) + ", " + num(l.lanes) + ", " + num(l.vec) + ", " + num(l.each) + ", " +
                                (residual ? "true" : "false") + ">(" + a + ", " + (bits8(y.dt) ? (residual ? "a5" : "a3") : "(float*)0") + ", " + flt(c.number("eps", 1e-6)) + ");");
  const int64_t lines = l.lanes < 256 ? 256 / l.lanes : 1;
  k.grid[0] = (unsigned)std::min<int64_t>((rows + lines - 1) / lines, kMaxGrid);
  for (auto& t : s.in) k.bytes += (double)t.bytes();
  for (auto& t : s.out) k.bytes += (double)t.bytes();
  p.kernels.push_back(k);
  return p;
}

void check_norm_grad(const Checker& c) {
  const auto &in = c.s.in, &out = c.s.out;
  c.settings({"eps"});
  check_eps(c);
  const TType& h = in[0];
  c.floats(h, "h");
  c.require(h.rank() >= 1 && h.dims.back() >= 1 && h.dims.back() <= kMaxNorm, "rows of 1 to " + num(kMaxNorm) + " elements are supported, got " + h.str());
  c.dims(in[1], {h.dims.back()}, "the weight");
  c.require(in[1].dt == h.dt, "the weight must have the type of h");
  c.same(h, in[2], "h and dy");
  if (in.size() == 4) c.same(h, in[3], "h and dh");
  c.same(h, out[0], "h and dx");
  c.dims(out[1], in[1].dims, "dweight");
  c.require(out[1].dt == h.dt || out[1].dt == DT::F32, "dweight must have the type of h, or be f32");
  c.require(h.numel() / h.dims.back() <= kMaxRow, "too many rows");
}
OperatorPlan plan_norm_grad(const OperatorSpec& s, bool lean) {
  const Checker c{s};
  const bool residual = s.in.size() == 4;
  const int64_t D = s.in[0].dims.back(), rows = s.in[0].numel() / D;
  const Lanes l = lanes_of(D, info(s.in[0].dt).size);
  const int64_t lines = l.lanes < 256 ? 256 / l.lanes : 1, most = 512;   // (256, 512 and 1024 workgroups: 40960 x 1024 bf16 57, 54 and 57 us, 16384 x 4096 113, 89 and 93, 8192 x 8192 98, 90 and 92, 4096 x 16384 91, 95 and 102)
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>({(rows + lines - 1) / lines, most, lean ? std::max<int64_t>(1, kLeanBytes / (4 * D)) : most}));
  OperatorPlan p;
  p.header = "rx_lm_norm_kernels.h";
  p.scratch = {groups * D * 4};
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (size_t i = 0; i < s.in.size(); ++i) args.push_back({operand((int)i), st(s.in[i])});
  args.push_back({result(0), st(s.out[0])});
  args.push_back({scratch(0), "float"});
  OperatorKernel k = kernel(s, "rms_norm_grad", (unsigned)std::max<int64_t>(256, l.lanes), args, 2,
                            std::string("rx_rms_norm_grad<") + elem(s.in[0].dt) + ", " + num(D) + ", " + num(rows) + ", " + num(l.lanes) + ", " + num(l.vec) + ", " + num(l.each) + ", " +
                                (residual ? "true" : "false") + ", " + num(groups) + ">(a0, a1, a2, " + (residual ? "a3, a4, a5" : "(" + st(s.in[0]) + "*)0, a3, a4") + ", " +
                                flt(c.number("eps", 1e-6)) + ");");
  k.grid[0] = (unsigned)groups;
  for (auto& t : s.in) k.bytes += (double)t.bytes();
  k.bytes += (double)s.out[0].bytes();
  p.kernels.push_back(k);
  k = kernel(s, "rms_norm_weight", 1024, {{scratch(0), "float"}, {result(1), st(s.out[1])}}, 1,
             std::string("rx_rms_norm_weight<") + elem(s.out[1].dt) + ", " + num(D) + ", " + num(groups) + ">(a0, a1);");
  k.grid[0] = (unsigned)((D + (D % 4 ? 15 : 63)) / (D % 4 ? 16 : 64));
  k.bytes = (double)s.out[1].bytes();
  p.kernels.push_back(k);
  return p;
}

// ------------------------------------------------------------------ caches
void check_write(const Checker& c) {
  const auto &in = c.s.in, &out = c.s.out;
  c.settings({"rotation", "layout", "sections"});
  const std::string rotation = c.word("rotation", "halves", {"halves", "pairs", "none"});
  const bool by_slot = by_slots(c);
  for (int i = 0; i < 3; ++i) {
    c.rank(in[i], 3, i == 0 ? "q" : i == 1 ? "k" : "v");
    c.floats(in[i], i == 0 ? "q" : i == 1 ? "k" : "v");
    c.require(in[i].dt == in[0].dt, "q, k and v must have one type");
  }
  check_stored(c, 9, 8, by_slot, in[0].dt);
  const Cache kc(in[9], by_slot), vc(in[10], by_slot);
  const int64_t T = in[0].dims[0];
  c.dims(in[0], {T, in[0].dims[1], kc.dim}, "q");
  c.dims(in[1], {T, kc.heads, kc.dim}, "k");
  c.dims(in[2], {T, kc.heads, vc.dim}, "v");
  c.f32(in[3], "cos");
  c.same(in[3], in[4], "cos and sin");
  c.rank(in[3], 2, "cos");
  c.require(in[3].dims[0] <= kMaxRow, "too many positions");
  c.require(rotation == "none" || 2 * in[3].dims[1] <= kc.dim, "the rotated dimensions exceed the head's: " + in[3].str() + " for heads of " + num(kc.dim));
  c.rank(in[5], 2, "angle");
  c.ints(in[5], "angle");
  const int64_t axes = in[5].dims[0];
  c.require(axes >= 1 && axes <= 4, "one to four axes are supported, got " + num(axes));
  c.dims(in[5], {axes, T}, "angle");
  sections_of(c, axes, in[3].dims[1]);
  c.ints(in[6], "position");
  c.dims(in[6], {T}, "position");
  c.same(in[6], in[7], "position and sequence");
  c.require(in[8].dt == in[6].dt && in[5].dt == in[6].dt, "angle, position, sequence and the page table must have one type");
  c.require(out.size() == in.size() - 8, "wrong number of results: " + num((int64_t)out.size()));
  c.same(out[0], in[0], "q and its result");
  for (size_t r = 1; r < out.size(); ++r) c.same(out[r], in[8 + r], r == 1 ? "k_cache and its result" : r == 2 ? "v_cache and its result" : r == 3 ? "k_scale and its result" : "v_scale and its result");
  c.require(T <= kMaxRow && in[0].dims[1] <= (1 << 20), "too many tokens or heads");
}
OperatorPlan plan_write(const OperatorSpec& s) {
  const Checker c{s};
  const auto& in = s.in;
  const bool by_slot = by_slots(c), scales = in.size() == 13;
  const std::string rotation = c.word("rotation", "halves", {"halves", "pairs", "none"});
  const Cache kc(in[9], by_slot), vc(in[10], by_slot);
  const int64_t T = in[0].dims[0], HQ = in[0].dims[1], R2 = rotation == "none" ? 0 : in[3].dims[1], axes = R2 ? in[5].dims[0] : 1;
  std::vector<int64_t> ends{0, 0, 0};
  const std::vector<int64_t> sections = sections_of(c, in[5].dims[0], in[3].dims[1]);
  for (int64_t a = 0, end = 0; a < axes && a < 3; ++a) ends[a] = end += sections[a];
  OperatorPlan p;
  p.header = "rx_lm_cache_kernels.h";
  p.updates = {-1, 9, 10};
  if (scales) p.updates.insert(p.updates.end(), {11, 12});
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < 9; ++i) args.push_back({operand(i), st(in[i])});
  for (size_t r = 0; r < s.out.size(); ++r) args.push_back({result((int)r), cell(s.out[r])});
  const int64_t ne = 16 / info(in[0].dt).size;
  const bool pairs = rotation == "pairs", whole = kc.dim % ne == 0 && vc.dim % ne == 0 && 2 * R2 % ne == 0 && (pairs || R2 % ne == 0);
  int64_t lanes = 1;
  while (lanes * ne < std::max(kc.dim, vc.dim)) lanes *= 2;
  // heads of a token to a group of lanes: 8191 tokens of 48 heads 41.3 us with two, 38.6 with four, 48.4 with eight; with one and with four 256 tokens 4.8 and 7.4 us,
  // 1024 9.8 and 10.3, 2048 16.5 and 14.0, 4096 28 and 23; 48 tokens 3.4 with one
  const int64_t each = T >= 2048 ? 4 : 1;
  std::ostringstream b;
  b << "rx_kv_write<" << elem(in[0].dt) << ", " << stored(in[9].dt) << ", " << HQ << ", " << kc.heads << ", " << kc.dim << ", " << vc.dim << ", " << kc.pages << ", " << kc.slots << ", "
    << in[8].dims[0] << ", " << in[8].dims[1] << ", " << in[3].dims[0] << ", " << R2 << ", " << axes << ", " << ends[0] << ", " << ends[1] << ", " << ends[2] << ", " << (pairs ? "true" : "false") << ", "
    << (by_slot ? "true" : "false") << ", " << T << ", " << (whole ? "true" : "false") << ", " << each << ">(a0, a1, a2, a3, a4, a5, a6, a7, a8, a9, a10, a11, "
    << (scales ? "a12, a13" : "(float*)0, (float*)0") << ");";
  OperatorKernel k = kernel(s, "kv_write", 256, args, (int)s.out.size(), b.str());
  const int64_t groups = (HQ + each - 1) / each + 2 * ((kc.heads + each - 1) / each);
  k.grid[0] = (unsigned)std::min<int64_t>((T * groups * lanes + 255) / 256, kMaxGrid);
  const double e = info(in[9].dt).size;
  k.bytes = 2.0 * (double)in[0].bytes() + (double)(in[1].bytes() + in[2].bytes()) + (double)(T * kc.heads) * ((double)(kc.dim + vc.dim) * e + (scales ? 8 : 0)) + 8.0 * (double)(T * R2) +
            (double)(in[6].bytes() * (2 + axes));
  p.kernels.push_back(k);
  return p;
}

void check_move(const Checker& c) {
  const auto &in = c.s.in, &out = c.s.out;
  c.settings({"layout"});
  check_stored(c, 3, 2, by_slots(c), DT::INVALID);
  c.rank(in[0], 1, "lengths");
  c.ints(in[0], "lengths");
  const int64_t B = in[0].dims[0];
  c.rank(in[1], 2, "path");
  c.require(in[1].dt == in[0].dt && in[2].dt == in[0].dt, "lengths, path and the page table must have one type");
  c.dims(in[1], {B, in[1].dims[1]}, "path");
  c.require(in[1].dims[1] <= kMaxSteps, "at most " + num(kMaxSteps) + " steps can be moved, got " + num(in[1].dims[1]));
  c.dims(in[2], {B, in[2].dims[1]}, "the page table");
  c.require(out.size() == in.size() - 3, "wrong number of results: " + num((int64_t)out.size()));
  for (size_t r = 0; r < out.size(); ++r) c.same(out[r], in[3 + r], r == 0 ? "k_cache and its result" : r == 1 ? "v_cache and its result" : r == 2 ? "k_scale and its result" : "v_scale and its result");
  c.require(B <= kMaxRow, "too many sequences");
}
OperatorPlan plan_move(const OperatorSpec& s) {
  const Checker c{s};
  const auto& in = s.in;
  const bool by_slot = by_slots(c), scales = in.size() == 7;
  const Cache kc(in[3], by_slot), vc(in[4], by_slot);
  const int64_t B = in[0].dims[0], A = in[1].dims[1], e = info(in[3].dt).size;
  // bytes of a unit: as many as divide the heads' rows, and as a thread's registers hold for all steps
  int64_t unit = A <= 16 ? 16 : A <= 32 ? 8 : 4;
  while ((kc.dim * e) % unit || (vc.dim * e) % unit) unit /= 2;
  const std::string word = unit == 16 ? "rx_u32x4" : unit == 8 ? "rx_u32x2" : unit == 4 ? "rx_u32" : unit == 2 ? "rx_u16" : "rx_u8";
  OperatorPlan p;
  p.header = "rx_lm_cache_kernels.h";
  p.updates = {3, 4};
  if (scales) p.updates.insert(p.updates.end(), {5, 6});
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < 3; ++i) args.push_back({operand(i), st(in[i])});
  for (size_t r = 0; r < s.out.size(); ++r) args.push_back({result((int)r), r < 2 ? word : std::string("float")});
  const int64_t ku = kc.dim * e / unit, vu = vc.dim * e / unit, units = kc.heads * (ku + vu + (scales ? 2 : 0));
  std::ostringstream b;
  b << "rx_kv_move<" << word << ", " << ku << ", " << vu << ", " << kc.heads << ", " << kc.pages << ", " << kc.slots << ", " << B << ", " << in[2].dims[1] << ", " << A << ", "
    << (by_slot ? "true" : "false") << ", " << (scales ? "true" : "false") << ">(a0, a1, a2, a3, a4, " << (scales ? "a5, a6" : "(float*)0, (float*)0") << ");";
  OperatorKernel k = kernel(s, "kv_move", 256, args, (int)s.out.size(), b.str());
  k.grid[0] = (unsigned)(A == 0 ? 0 : std::min<int64_t>((B * units + 255) / 256, kMaxGrid));
  k.bytes = 2.0 * (double)(B * A * units * unit);
  p.kernels.push_back(k);
  return p;
}

// ------------------------------------------------------------------ attention of drafted tokens
namespace {
int64_t pow2(int64_t n) {
  int64_t p = 1;
  while (p < n) p *= 2;
  return p;
}
// which operand is the mask (0: none), and the first of the scales (0: none)
int mask_of(const OperatorSpec& s) { return s.in.size() % 2 == 0 ? 5 : 0; }
int scales_of(const OperatorSpec& s) { return s.in.size() >= 7 ? (int)s.in.size() - 2 : 0; }
}  // namespace
void check_tree(const Checker& c) {
  const auto& in = c.s.in;
  c.settings({"scale", "window", "layout"});
  const bool by_slot = by_slots(c);
  c.rank(in[0], 4, "q");
  c.floats(in[0], "q");
  OperatorSpec some = c.s;          // the operands without the mask between them
  some.in = {in[3], in[1], in[2]};
  if (scales_of(c.s)) some.in.insert(some.in.end(), in.end() - 2, in.end());
  check_stored(Checker{some}, 1, 0, by_slot, in[0].dt);
  const Cache kc(in[1], by_slot), vc(in[2], by_slot);
  const int64_t B = in[0].dims[0], N = in[0].dims[1], Hq = in[0].dims[2];
  c.require(in[0].dims[3] == kc.dim, "q and k_cache must have the same head dimension");
  c.require(Hq >= 1 && Hq % kc.heads == 0, "the query heads (" + num(Hq) + ") must be a multiple of the cache's (" + num(kc.heads) + ")");
  c.require(N <= 1024, "at most 1024 drafted tokens are supported, got " + num(N));
  c.dims(in[3], {B, in[3].dims[1]}, "the page table");
  c.ints(in[4], "lengths");
  c.dims(in[4], {B}, "lengths");
  c.require(in[4].dt == in[3].dt, "lengths and the page table must have one type");
  if (const int m = mask_of(c.s)) {
    c.require(in[m].dt == DT::I1, "the mask must be i1, got " + in[m].str());
    c.require(in[m].dims == std::vector<int64_t>({N, N}) || in[m].dims == std::vector<int64_t>({B, N, N}), "the mask must be [" + num(N) + ", " + num(N) + "] or [" + num(B) + ", " + num(N) + ", " + num(N) + "], got " + in[m].str());
  }
  c.dims(c.s.out[0], {B, N, Hq, vc.dim}, "the result");
  c.require(c.s.out[0].dt == in[0].dt, "the result must have the type of q");
  if (c.s.out.size() == 2) {
    c.f32(c.s.out[1], "lse");
    c.dims(c.s.out[1], {B, N, Hq}, "lse");
  }
  c.scale(1.4426950408889634);
  const int64_t window = c.integer("window", 0);
  c.require(window == 0 || window >= N, "the window must hold the " + num(N) + " drafted tokens, or be 0 for none");
  c.require(window >= 0, "the window must not be negative");
  c.require(B <= 65535 && Hq <= 65535, "too many sequences or heads");
  c.require(B * N * Hq * std::max<int64_t>(vc.dim, kc.dim) <= kMaxRow, "too many sequences, drafted tokens and heads");
}
OperatorPlan plan_tree(const OperatorSpec& s, bool lean) {
  const Checker c{s};
  const auto& in = s.in;
  const bool by_slot = by_slots(c);
  const Cache kc(in[1], by_slot), vc(in[2], by_slot);
  const int64_t B = in[0].dims[0], N = in[0].dims[1], Hq = in[0].dims[2], M = in[3].dims[1], G = Hq / kc.heads, rows = N * G;
  const double scale = c.number("scale", 1.0 / std::sqrt((double)kc.dim));
  const int64_t window = std::min<int64_t>(c.integer("window", 0), kMaxRow);
  const bool lse = s.out.size() == 2, q8 = bits8(in[1].dt);
  const int mask = mask_of(s), scales = scales_of(s);
  OperatorPlan p;
  p.header = "rx_lm_cache_kernels.h";
  if (B * rows == 0) return p;
  const int64_t e = info(in[1].dt).size, qe = info(in[0].dt).size;
  const bool wide = !q8 && qe == 4;
  const int64_t fe = wide ? 4 : 8, size = wide ? 4 : 2, nq = !q8 ? 1 : qe == 4 ? 3 : in[0].dt == DT::F16 ? 2 : 1;
  const int64_t ve = wide || vc.dim <= 64 ? 4 : 8, nv = (vc.dim + 16 * ve - 1) / (16 * ve);
  // Up to 32 rows the wavefronts share the positions; more rows share keys and values through LDS, 64 or 128 to a workgroup (64 rows as two tiles of 32
  // that share positions: 218 us and more against 125, 512 as sixteen 555 against 380; 64 rows as half of 128: 178 against 125).
  const bool shared = rows > 32;
  // rows of whole 16 bytes: keys and values pass through a ring of stages, as many as leave room for a second workgroup
  const int64_t ce = 16 / e, places_k = std::max<int64_t>(4, pow2((kc.dim + ce - 1) / ce)), places_v = std::max<int64_t>(4, pow2((vc.dim + ce - 1) / ce)), stage = 512 * (places_k + places_v);
  const bool rings = shared && kc.dim % ce == 0 && vc.dim % ce == 0 && (places_k + places_v) % 8 == 0;
  const int64_t ring = !rings ? 0 : stage <= 16384 ? 4 : 2;   // (of 8 KB 3, 4 and 6: 120, 119 and 121 us for 64 sequences of 16 drafted tokens; of 16 KB 3 and 4: 383, 387)
  const int64_t kf = q8 && (!shared || rings) ? 2 * ((kc.dim + 63) / 64) : (kc.dim + 4 * fe - 1) / (4 * fe);
  // registers of a wavefront: a step's keys and values (and in many rows' case the next one's), the queries, the result, and room for the rest
  auto registers = [&](int64_t n) {
    const int64_t staged = shared && !rings ? ((32 * kc.dim * e + 4095) / 4096 + (32 * vc.dim * e + 4095) / 4096) * 4 : 0;
    return 8 * kf + 8 * nv * ve * size / 4 + staged + n * (4 * nq * kf + 4 * nv * ve + 24);
  };
  int64_t NT = 1;
  if (shared) NT = rows > 64 && registers(2) < 330 ? 2 : 1;
  else NT = rows > 16 && registers(2) < 320 ? 2 : 1;
  const int64_t WR = shared ? 4 : 1, TR = 16 * NT * WR, tiles = (rows + TR - 1) / TR, RT = std::min(rows, TR);
  const int64_t results = 64 * (16 * ve + 4) * 4;   // of four wavefronts' 16 rows
  const int64_t lds = rings ? std::max(ring * stage, results) + 4096 : shared ? 2 * 32 * ((kf * 4 * fe + 16 / size) + (nv * 16 * ve + 16 / size)) * size + results : 0;
  // Two wavefronts to a SIMD where the estimate says that they fit.  With one and with two, 16 sequences of 4000 positions, 8 key heads, bf16 unless said otherwise:
  // an estimate of 208, 8 and 32 rows of 128 dimensions 54 and 57 us, 60 and 63 (one sequence of 1000 positions 18.6 and 17.8); 212 to 224, 8 rows
  // of 160 and 192, 72 and 67, 84 and 84; 224, 64 rows of 192, 158 and 102; 240, 128 rows of 128, f16 over 8 bits, 157 and 127; 248, 64 rows of 256, 156 and 116; 256,
  // 32 rows of 80 in f32 115 and 108.  Beyond: 272, 32 rows of 128, f32 over 8 bits, 67 and 71; 280, 8 rows of 256, f16 over 8 bits, 77 and 90; 288, 8 rows
  // of 160 in f32 140 and 223; 304, 32 rows of 128 in f32 158 and 193.  (Four tiles of 16 rows to a wavefront, one to a SIMD: 614 where two take 380.)
  const int waves = registers(NT) <= 256 && lds <= 80000 ? 2 : 1;
  const int64_t longest = window ? std::min(M * kc.slots, window + N + 31) : M * kc.slots, units = std::max<int64_t>(1, (longest + 31) / 32);
  const bool once = kc.dim * e % 256 == 0 && vc.dim * e % 256 == 0 && tiles == 1, dies = (by_slot && kc.dim * e % 128 != 0) || tiles > 1;
  const int64_t columns = kc.heads * tiles, room = 256 * waves;
  // every workgroup a stretch of at least four units of 32 positions (a sequence counts four more), all of them on the chip at once
  const int64_t part = 2 * RT * (vc.dim * 4 + 8), most = lean ? std::min<int64_t>(room, kLeanBytes / part) : room;
  const int64_t stretches = std::max<int64_t>(1, std::min(most / columns, (B * (units + (B > 1 ? 4 : 0)) + 3) / 4)), grid = stretches * columns;
  std::vector<std::pair<OperatorArg, std::string>> args;
  for (int i = 0; i < (int)in.size(); ++i) args.push_back({operand(i), i == 1 || i == 2 ? cell(in[i]) : st(in[i])});
  for (int r = 0; r < (int)s.out.size(); ++r) args.push_back({result(r), st(s.out[r])});
  auto a = [](int i) { return "a" + num(i); };
  const int o = (int)in.size();
  std::string shared_args = "(float*)0, (float*)0, (int*)0";
  if (stretches > 1) {
    p.scratch = {grid * 2 * RT * vc.dim * 4, grid * 2 * RT * 8};
    p.counters = B * columns;
    const int at = (int)args.size();
    args.push_back({scratch(0), "float"});
    args.push_back({scratch(1), "float"});
    args.push_back({counters(), "int"});
    shared_args = a(at) + ", " + a(at + 1) + ", " + a(at + 2);
  }
  std::ostringstream b;
  b << "rx_tree_attention<" << elem(in[0].dt) << ", " << stored(in[1].dt) << ", " << N << ", " << Hq << ", " << kc.heads << ", " << kc.dim << ", " << vc.dim << ", " << kc.pages << ", " << kc.slots << ", "
    << B << ", " << M << ", " << window << ", " << (by_slot ? "true" : "false") << ", " << (mask ? in[mask].rank() : 0) << ", " << NT << ", " << WR << ", " << ring << ", " << stretches << ", "
    << (once ? "true" : "false") << ", " << (dies ? "true" : "false") << ", " << std::max<int64_t>(1, std::min<int64_t>(4, 4096 / (RT * vc.dim))) << ">(a0, a1, a2, a3, a4, "
    << (mask ? a(mask) : "(rx_u8*)0") << ", " << (scales ? a(scales) + ", " + a(scales + 1) : "(float*)0, (float*)0") << ", " << a(o) << ", " << (lse ? a(o + 1) : "(float*)0") << ", " << shared_args
    << ", " << flt(scale * 1.4426950408889634) << ");";
  OperatorKernel k = kernel(s, "tree_attention", 256, args, (int)args.size() - o, b.str(), waves);
  k.grid[0] = (unsigned)grid;
  k.bytes = (double)(in[0].bytes() + s.out[0].bytes());   // (and what the lengths make of the caches)
  p.kernels.push_back(k);
  return p;
}

double serve_flops(const OperatorSpec& s, double* transcendentals) {
  if (s.name == "rx.rms_norm") return 6.0 * (double)s.in[0].numel();
  if (s.name == "rx.rms_norm_grad") return 11.0 * (double)s.in[0].numel();
  if (s.name == "rx.kv_write") return 3.0 * 2.0 * (double)s.in[3].dims[1] * (double)(s.in[0].dims[0] * (s.in[0].dims[1] + s.in[1].dims[1]));
  if (s.name != "rx.tree_attention") return 0.0;
  const Checker c{s};
  const Cache kc(s.in[1], by_slots(c));   // the longest the page table allows
  const double n = (double)(s.in[3].dims[1] * kc.slots) * (double)(s.in[0].numel() / std::max<int64_t>(1, s.in[0].dims[3]));
  *transcendentals = n;
  return 2.0 * n * (double)(kc.dim + s.in[2].dims[3]);
}

}  // namespace lm
}  // namespace rx
