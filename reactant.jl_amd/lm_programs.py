"""Module text of the language-model operators: `stablehlo.custom_call` of the backend's `rx.` targets, and programs that
use them together.  Like programs.py this stands in for the tracing front end; a traced program holds the same calls
(`MLIR.Dialects.stablehlo.custom_call` with `call_target_name` and a `backend_config` dictionary, reference
src/mlir/Dialects/StableHLO.jl).

Each writer names its shapes in the module's row-major order and returns text for `compile`; what the targets compute is
stated in csrc/rx_lm.h.  Arguments come in the order of the operands.  Cache arguments are marked with the result that may
take them over: a call with them donated updates the caches in place, one without copies them first."""


EIGHT_BITS = ("f8E4M3FN", "i8")     # types of numbers that stand for their product with a scale


def tt(shape, dt):
    return "tensor<" + "".join("%dx" % d for d in shape) + dt + ">"


def _config(settings):
    """`backend_config`: numbers and strings; None is left out."""
    out = []
    for key, value in settings.items():
        if value is None:
            continue
        if isinstance(value, str):
            out.append('%s = "%s"' % (key, value))
        elif isinstance(value, float):
            out.append("%s = %.17e : f64" % (key, value))
        else:
            out.append("%s = %d : i64" % (key, value))
    return "{" + ", ".join(out) + "}"


def custom_call(target, operands, types, results, settings=None, name="%0"):
    """One line: `name` = the operator on SSA `operands` of `types`, giving `results` (types)."""
    lhs = name + (":%d" % len(results) if len(results) > 1 else "")
    rt = results[0] if len(results) == 1 else "(" + ", ".join(results) + ")"
    return ("    %s = stablehlo.custom_call @%s(%s) {api_version = 4 : i32, backend_config = %s} : (%s) -> %s\n"
            % (lhs, target, ", ".join(operands), _config(settings or {}), ", ".join(types), rt))


def _module(name, target, args, results, settings=None, aliases=None):
    """A function that is one operator.  `aliases`: argument -> result that may take it over."""
    aliases = aliases or {}
    params = ", ".join("%%arg%d: %s%s" % (k, t, " {tf.aliasing_output = %d : i32}" % aliases[k] if k in aliases else "")
                       for k, t in enumerate(args))
    names = ["%0"] if len(results) == 1 else ["%%0#%d" % k for k in range(len(results))]
    rt = results[0] if len(results) == 1 else "(" + ", ".join(results) + ")"
    return ("module @reactant_%s {\n  func.func @main(%s) -> %s {\n" % (name, params, rt)
            + custom_call(target, ["%%arg%d" % k for k in range(len(args))], args, results, settings)
            + "    return %s : %s\n  }\n}\n" % (", ".join(names), ", ".join(results)))


def embedding(tokens, rows, width, dt="bf16", ids="i32", scale=1.0):
    """(table [rows, width], ids [tokens]) -> [tokens, width]: scaled rows, zeros for tokens outside of the table."""
    return _module("embedding", "rx.embedding", [tt([rows, width], dt), tt([tokens], ids)], [tt([tokens, width], dt)], {"scale": float(scale)})


def embedding_grad(tokens, rows, width, dt="bf16", out=None, ids="i32", scale=1.0):
    """(dy [tokens, width], ids [tokens]) -> the table's gradient [rows, width] in type `out` (dt or f32)."""
    return _module("embedding_grad", "rx.embedding_grad", [tt([tokens, width], dt), tt([tokens], ids)], [tt([rows, width], out or dt)], {"scale": float(scale)})


def cache_shape(num_pages, page_size, kv_heads, head_dim, layout="slots"):
    return [num_pages, page_size, kv_heads, head_dim] if layout == "slots" else [num_pages, kv_heads, page_size, head_dim]


def kv_append(tokens, sequences, q_heads, kv_heads, head_dim, num_pages, page_size, table_pages, positions, dt="bf16", rotary_dim=None,
              rotation="halves", layout="slots", ids="i32", value_dim=None):
    """(q, k, v, cos, sin, position, sequence, page table, k_cache, v_cache) -> (rotated q, k_cache, v_cache).  `positions` rows
    of the cosine and sine tables [positions, rotary_dim / 2]; donate the caches to update them in place."""
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    value_dim = value_dim or head_dim
    kc, vc = (tt(cache_shape(num_pages, page_size, kv_heads, d, layout), dt) for d in (head_dim, value_dim))
    q = tt([tokens, q_heads, head_dim], dt)
    angles, index = tt([positions, rotary_dim // 2], "f32"), tt([tokens], ids)
    args = [q, tt([tokens, kv_heads, head_dim], dt), tt([tokens, kv_heads, value_dim], dt), angles, angles, index, index,
            tt([sequences, table_pages], ids), kc, vc]
    return _module("kv_append", "rx.kv_append", args, [q, kc, vc], {"rotation": rotation, "layout": layout}, {8: 1, 9: 2})


def paged_attention(sequences, q_heads, kv_heads, head_dim, num_pages, page_size, table_pages, dt="bf16", scale=None, window=0, layout="slots",
                    ids="i32", value_dim=None, lse=False):
    """(q [sequences, q_heads, head_dim], k_cache, v_cache, page table, lengths) -> attention of one token per sequence, and
    with `lse` the log of its sums of exponentials.  `scale`: 1 / sqrt(head_dim) if not given; `window`: the last positions only."""
    value_dim = value_dim or head_dim
    kc, vc = (tt(cache_shape(num_pages, page_size, kv_heads, d, layout), dt) for d in (head_dim, value_dim))
    res = [tt([sequences, q_heads, value_dim], dt)] + ([tt([sequences, q_heads], "f32")] if lse else [])
    return _module("paged_attention", "rx.paged_attention", [tt([sequences, q_heads, head_dim], dt), kc, vc, tt([sequences, table_pages], ids), tt([sequences], ids)], res,
                   {"scale": None if scale is None else float(scale), "window": window, "layout": layout})


def token_logprobs(tokens, vocab, top=0, dt="bf16", ids="i32"):
    """(logits [tokens, vocab], targets [tokens]) -> (logprob, lse, entropy) in f32, and with `top` the largest log
    probabilities [tokens, top] and their indices (i32)."""
    one = tt([tokens], "f32")
    res = [one, one, one] + ([tt([tokens, top], "f32"), tt([tokens, top], "i32")] if top else [])
    return _module("token_logprobs", "rx.token_logprobs", [tt([tokens, vocab], dt), tt([tokens], ids)], res, {"top": top})


def token_logprobs_grad(tokens, vocab, dt="bf16", ids="i32"):
    """(logits, targets, lse, entropy, d_logprob, d_entropy) -> gradient of the logits."""
    one = tt([tokens], "f32")
    logits = tt([tokens, vocab], dt)
    return _module("token_logprobs_grad", "rx.token_logprobs_grad", [logits, tt([tokens], ids), one, one, one, one], [logits])


def rms_norm(rows, width, dt="bf16", out=None, eps=1e-6, residual=True):
    """(x [rows, width] [, residual], weight [width]) -> ([h = x + residual,] norm of h times weight in type `out`).  `out` of 8 bits
    (f8E4M3FN or i8) gives the rows' scales [rows] as one more result.  Without residual and 8 bits the same as a reduction in the traced
    program is one launch too, and a faster one, most of all for rows of a head's few dimensions."""
    x, out = tt([rows, width], dt), out or dt
    res = ([x] if residual else []) + [tt([rows, width], out)] + ([tt([rows], "f32")] if out in EIGHT_BITS else [])
    return _module("rms_norm", "rx.rms_norm", [x, x, tt([width], dt)] if residual else [x, tt([width], dt)], res, {"eps": float(eps)})


def rms_norm_grad(rows, width, dt="bf16", out="f32", eps=1e-6, residual=True):
    """(h [rows, width], weight [width], dy [, dh]) -> (gradient by h, gradient by weight in type `out`, f32 or dt)."""
    x, w = tt([rows, width], dt), tt([width], dt)
    return _module("rms_norm_grad", "rx.rms_norm_grad", [x, w, x, x] if residual else [x, w, x], [x, tt([width], out)], {"eps": float(eps)})


def _caches(num_pages, page_size, kv_heads, head_dim, value_dim, layout, cache):
    """Types of the caches, and of their scales where they hold 8 bits."""
    scale = tt([num_pages, kv_heads, page_size], "f32")
    return [tt(cache_shape(num_pages, page_size, kv_heads, d, layout), cache) for d in (head_dim, value_dim)] + ([scale, scale] if cache in EIGHT_BITS else [])


def kv_write(tokens, sequences, q_heads, kv_heads, head_dim, num_pages, page_size, table_pages, positions, dt="bf16", cache=None, sections=None, rotary_dim=None,
             rotation="halves", layout="slots", ids="i32", value_dim=None):
    """(q, k, v, cos, sin, angle [axes, tokens], position, sequence, page table, k_cache, v_cache [, k_scale, v_scale]) -> (rotated q, the
    caches and their scales).  `sections`: rotated pairs that follow each axis' angles (one axis if not given); `cache`: the caches' type,
    dt or of 8 bits, which have scales.  Donate the caches to update them in place."""
    rotary_dim = (2 * sum(sections) if sections else head_dim) if rotary_dim is None else rotary_dim
    value_dim, axes = value_dim or head_dim, len(sections) if sections else 1
    stored = _caches(num_pages, page_size, kv_heads, head_dim, value_dim, layout, cache or dt)
    q, angles, index = tt([tokens, q_heads, head_dim], dt), tt([positions, rotary_dim // 2], "f32"), tt([tokens], ids)
    args = [q, tt([tokens, kv_heads, head_dim], dt), tt([tokens, kv_heads, value_dim], dt), angles, angles, tt([axes, tokens], ids), index, index,
            tt([sequences, table_pages], ids)] + stored
    return _module("kv_write", "rx.kv_write", args, [q] + stored,
                   {"rotation": rotation, "layout": layout, "sections": ",".join(map(str, sections)) if sections else None}, {9 + i: 1 + i for i in range(len(stored))})


def kv_move(sequences, steps, kv_heads, head_dim, num_pages, page_size, table_pages, cache="bf16", layout="slots", ids="i32", value_dim=None):
    """(lengths [sequences], path [sequences, steps], page table, k_cache, v_cache [, k_scale, v_scale]) -> the caches, where position
    lengths + i holds what position lengths + path[i] held.  Donate the caches to update them in place."""
    stored = _caches(num_pages, page_size, kv_heads, head_dim, value_dim or head_dim, layout, cache)
    return _module("kv_move", "rx.kv_move", [tt([sequences], ids), tt([sequences, steps], ids), tt([sequences, table_pages], ids)] + stored, stored, {"layout": layout},
                   {3 + i: i for i in range(len(stored))})


def tree_attention(sequences, drafted, q_heads, kv_heads, head_dim, num_pages, page_size, table_pages, dt="bf16", cache=None, mask=True, scale=None, window=0, layout="slots",
                   ids="i32", value_dim=None, lse=False):
    """(q [sequences, drafted, q_heads, head_dim], k_cache, v_cache, page table, lengths [, mask] [, k_scale, v_scale]) -> attention of the
    drafted tokens, which lie behind the first `lengths` positions of the cache.  `mask`: True for one [drafted, drafted] per sequence,
    "shared" for one of all, False for none: a token then sees itself and those before it."""
    value_dim = value_dim or head_dim
    stored = _caches(num_pages, page_size, kv_heads, head_dim, value_dim, layout, cache or dt)
    q = [sequences, drafted, q_heads]
    args = [tt(q + [head_dim], dt), stored[0], stored[1], tt([sequences, table_pages], ids), tt([sequences], ids)]
    args += [tt(([] if mask == "shared" else [sequences]) + [drafted, drafted], "i1")] if mask else []
    return _module("tree_attention", "rx.tree_attention", args + stored[2:], [tt(q + [value_dim], dt)] + ([tt(q, "f32")] if lse else []),
                   {"scale": None if scale is None else float(scale), "window": window, "layout": layout})


# ----------------------------------------------------------------------------
# the operators together
# ----------------------------------------------------------------------------
class _Text:
    """Lines of a function body, with the type of every value."""

    def __init__(self):
        self.lines, self.types, self.shapes, self.args, self.n = [], {}, {}, [], 0

    def arg(self, shape, dt, alias=None):
        name = "%%arg%d" % len(self.args)
        self.types[name], self.shapes[name] = tt(shape, dt), (list(shape), dt)
        self.args.append("%s: %s%s" % (name, tt(shape, dt), "" if alias is None else " {tf.aliasing_output = %d : i32}" % alias))
        return name

    def op(self, text, shape, dt):
        self.n += 1
        name = "%%v%d" % self.n
        self.types[name], self.shapes[name] = tt(shape, dt), (list(shape), dt)
        self.lines.append("    %s = stablehlo.%s -> %s\n" % (name, text, tt(shape, dt)))
        return name

    def binary(self, op, a, b):
        return self.op("%s %s, %s : (%s, %s)" % (op, a, b, self.types[a], self.types[b]), *self.shapes[a])

    def select(self, where, a, b):
        self.n += 1
        name = "%%v%d" % self.n
        self.types[name], self.shapes[name] = self.types[a], self.shapes[a]
        self.lines.append("    %s = stablehlo.select %s, %s, %s : %s, %s\n" % (name, where, a, b, self.types[where], self.types[a]))
        return name

    def constant(self, literal, shape, dt):
        self.n += 1
        name = "%%c%d" % self.n
        self.types[name], self.shapes[name] = tt(shape, dt), (list(shape), dt)
        self.lines.append("    %s = stablehlo.constant dense<%s> : %s\n" % (name, literal, tt(shape, dt)))
        return name

    def iota(self, n, dim=0):
        """0, 1, .. along a dimension of `n` (a size, or several)."""
        shape = list(n) if isinstance(n, (list, tuple)) else [n]
        self.n += 1
        name = "%%v%d" % self.n
        self.types[name], self.shapes[name] = tt(shape, "i32"), (shape, "i32")
        self.lines.append("    %s = stablehlo.iota dim = %d : %s\n" % (name, dim, tt(shape, "i32")))
        return name

    def convert(self, x, dt):
        return x if self.shapes[x][1] == dt else self.op("convert %s : (%s)" % (x, self.types[x]), self.shapes[x][0], dt)

    def reshape(self, x, shape):
        return self.op("reshape %s : (%s)" % (x, self.types[x]), shape, self.shapes[x][1])

    def spread(self, x, dims, shape):
        return self.op("broadcast_in_dim %s, dims = %s : (%s)" % (x, dims, self.types[x]), shape, self.shapes[x][1])

    def dot(self, a, b, dims, dt=None):
        """Product over one dimension of each ([i] x [j] of matrices)."""
        (sa, ta), (sb, _) = self.shapes[a], self.shapes[b]
        shape = [sa[1 - dims[0]], sb[1 - dims[1]]]
        return self.op("dot_general %s, %s, contracting_dims = [%d] x [%d], precision = [DEFAULT, DEFAULT] : (%s, %s)"
                       % (a, b, dims[0], dims[1], self.types[a], self.types[b]), shape, dt or ta)

    def operator(self, target, operands, results, settings=None):
        self.n += 1
        name = "%%v%d" % self.n
        names = [name] if len(results) == 1 else ["%s#%d" % (name, k) for k in range(len(results))]
        for k, r in zip(names, results):
            self.types[k], self.shapes[k] = tt(*r), (list(r[0]), r[1])
        self.lines.append(custom_call(target, operands, [self.types[o] for o in operands], [tt(*r) for r in results], settings, name))
        return names

    def rms_norm(self, x, weight):
        """x / sqrt(mean(x^2) + 1e-6) * weight, in f32."""
        (n, w), dt = self.shapes[x]
        f = self.convert(x, "f32")
        sq = self.binary("multiply", f, f)
        zero = self.constant("0.000000e+00", [], "f32")
        total = self.op("reduce(%s init: %s) applies stablehlo.add across dimensions = [1] : (%s, tensor<f32>)" % (sq, zero, self.types[sq]), [n], "f32")
        mean = self.binary("multiply", total, self.constant("%.9e" % (1.0 / w), [n], "f32"))
        mean = self.binary("add", mean, self.constant("1.000000e-06", [n], "f32"))
        root = self.op("rsqrt %s : (%s)" % (mean, self.types[mean]), [n], "f32")
        y = self.binary("multiply", f, self.spread(root, [0], [n, w]))
        return self.convert(self.binary("multiply", y, self.spread(self.convert(weight, "f32"), [1], [n, w])), dt)

    def module(self, name, results):
        rt = ", ".join(self.types[r] for r in results)
        return ("module @reactant_%s {\n  func.func @main(%s) -> (%s) {\n" % (name, ", ".join(self.args), rt) + "".join(self.lines)
                + "    return %s : %s\n  }\n}\n" % (", ".join(results), rt))


def decode_step(sequences, vocab, width, q_heads, kv_heads, head_dim, hidden, num_pages, page_size, table_pages, positions, layers=1, top=5,
                dt="bf16", layout="slots", rotation="halves"):
    """One token of every sequence through a transformer with paged caches: embedding, then per layer norm, attention over the
    cache that the token's key and value have been appended to, norm and a gated MLP, then the log probabilities over the
    vocabulary.  Returns (text, [(shape, element type)] of the arguments, results that are caches): arguments are tokens, targets,
    position, page table, cos, sin, embedding table, per layer (norm, wq, wk, wv, wo, norm, gate, up, down, k_cache, v_cache), norm
    and head; results are (logprob, lse, entropy, top log probabilities, top indices) and the caches, which the cache arguments
    may be donated to.  A sequence whose position is -1 takes no part."""
    b, x = sequences, _Text()
    tokens, targets, position = (x.arg([b], "i32") for _ in range(3))
    pages = x.arg([b, table_pages], "i32")
    cos, sin = (x.arg([positions, head_dim // 2], "f32") for _ in range(2))
    table = x.arg([vocab, width], dt)
    first_cache = 5
    weights = []
    for l in range(layers):
        w = {"norm1": x.arg([width], dt)}
        for key, heads in (("q", q_heads), ("k", kv_heads), ("v", kv_heads)):
            w[key] = x.arg([width, heads * head_dim], dt)
        w["o"], w["norm2"] = x.arg([q_heads * head_dim, width], dt), x.arg([width], dt)
        w["gate"], w["up"], w["down"] = x.arg([width, hidden], dt), x.arg([width, hidden], dt), x.arg([hidden, width], dt)
        shape = cache_shape(num_pages, page_size, kv_heads, head_dim, layout)
        w["k_cache"], w["v_cache"] = (x.arg(shape, dt, first_cache + 2 * l + k) for k in range(2))
        weights.append(w)
    norm, head = x.arg([width], dt), x.arg([width, vocab], dt)
    sequence = x.iota(b)
    lengths = x.binary("add", position, x.constant("1", [b], "i32"))
    h = x.operator("rx.embedding", [table, tokens], [([b, width], dt)], {"scale": 1.0})[0]
    caches = []
    for w in weights:
        y = x.rms_norm(h, w["norm1"])
        q, k, v = (x.reshape(x.dot(y, w[key], (1, 0)), [b, heads, head_dim]) for key, heads in (("q", q_heads), ("k", kv_heads), ("v", kv_heads)))
        q, kc, vc = x.operator("rx.kv_append", [q, k, v, cos, sin, position, sequence, pages, w["k_cache"], w["v_cache"]],
                               [([b, q_heads, head_dim], dt), x.shapes[w["k_cache"]], x.shapes[w["v_cache"]]], {"rotation": rotation, "layout": layout})
        caches += [kc, vc]
        a = x.operator("rx.paged_attention", [q, kc, vc, pages, lengths], [([b, q_heads, head_dim], dt)], {"layout": layout})[0]
        h = x.binary("add", h, x.dot(x.reshape(a, [b, q_heads * head_dim]), w["o"], (1, 0)))
        y = x.rms_norm(h, w["norm2"])
        gate = x.dot(y, w["gate"], (1, 0))
        act = x.binary("multiply", gate, x.op("logistic %s : (%s)" % (gate, x.types[gate]), [b, hidden], dt))
        h = x.binary("add", h, x.dot(x.binary("multiply", act, x.dot(y, w["up"], (1, 0))), w["down"], (1, 0)))
    logits = x.dot(x.rms_norm(h, norm), head, (1, 0))
    one = ([b], "f32")
    out = x.operator("rx.token_logprobs", [logits, targets], [one, one, one, ([b, top], "f32"), ([b, top], "i32")], {"top": top})
    return x.module("decode_step", out + caches), [x.shapes["%%arg%d" % k] for k in range(len(x.args))], list(range(first_cache, first_cache + 2 * layers))


def verify_step(sequences, drafted, vocab, width, q_heads, kv_heads, head_dim, hidden, num_pages, page_size, table_pages, positions, layers=1, axes=1, top=5, dt="bf16",
                cache="f8E4M3FN", products="f8E4M3FN", layout="slots", rotation="halves"):
    """A tree of drafted tokens of every sequence through a transformer with paged caches: embedding, then per layer norm, keys and
    values written behind the sequence's positions (`cache`: their type), attention that the tree masks, sum with the residual and norm,
    a gated MLP, and the log probabilities of every token's successor.  The norms give 8 bits for the products that follow them
    (`products`: their type, that of the weights [outputs, inputs] there, whose factors are numbers; or dt).  With one drafted token
    this is a decoding step.  Returns (text, [(shape, element type)] of the arguments, results that are caches).  Arguments are tokens
    [sequences, drafted], targets (the successor that is asked about), angle [axes, sequences, drafted] (rows of the tables of angles),
    lengths (-1: takes no part), mask, page table, cos, sin, embedding table, per layer (norm, wq, wk, wv, wo, norm, gate, up, down,
    then the factors of wq, wk, wv, gate and up where the products have 8 bits, k_cache, v_cache and their scales), norm and head;
    results are (logprob, lse, entropy, top log probabilities, top indices) and the caches, which the cache arguments may be donated
    to.  `rx.kv_move` brings together what the accepted branch has written."""
    b, n, x = sequences, drafted, _Text()
    t, eight, stored = b * n, products in EIGHT_BITS, cache in EIGHT_BITS
    tokens, targets = (x.arg([b, n], "i32") for _ in range(2))
    angle, lengths, mask, pages = x.arg([axes, b, n], "i32"), x.arg([b], "i32"), x.arg([b, n, n], "i1"), x.arg([b, table_pages], "i32")
    cos, sin = (x.arg([positions, head_dim // 2], "f32") for _ in range(2))
    table = x.arg([vocab, width], dt)
    first_cache, held = 5, 4 if stored else 2
    weights = []
    for l in range(layers):
        w = {"norm1": x.arg([width], dt)}
        for key, heads in (("q", q_heads), ("k", kv_heads), ("v", kv_heads)):
            w[key] = x.arg([heads * head_dim, width], products)
        w["o"], w["norm2"] = x.arg([width, q_heads * head_dim], dt), x.arg([width], dt)
        w["gate"], w["up"], w["down"] = x.arg([hidden, width], products), x.arg([hidden, width], products), x.arg([width, hidden], dt)
        if eight:
            w["factor"] = {key: x.arg([], "f32") for key in ("q", "k", "v", "gate", "up")}
        shapes = [(cache_shape(num_pages, page_size, kv_heads, head_dim, layout), cache)] * 2 + [([num_pages, kv_heads, page_size], "f32")] * (held - 2)
        w["caches"] = [x.arg(*s, first_cache + held * l + k) for k, s in enumerate(shapes)]
        weights.append(w)
    norm, head = x.arg([width], dt), x.arg([vocab, width], dt)
    sequence = x.reshape(x.iota([b, n]), [t])
    base = x.spread(lengths, [0], [b, n])
    there = x.op("compare GE, %s, %s, SIGNED : (%s, %s)" % (base, x.constant("0", [b, n], "i32"), x.types[base], x.types[base]), [b, n], "i1")
    position = x.binary("add", base, x.iota([b, n], 1))
    position = x.select(there, position, x.constant("-1", [b, n], "i32"))
    position, angle = x.reshape(position, [t]), x.reshape(angle, [axes, t])
    half = head_dim // 2
    sections = [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)

    def normed(v, residual, weight, out):
        """([h,] norm, scale) of v [+ residual]."""
        rows = [([t, width], dt)] if residual else []
        res = rows + [([t, width], out)] + ([([t], "f32")] if out in EIGHT_BITS else [])
        got = x.operator("rx.rms_norm", [v] + ([residual] if residual else []) + [weight], res, {"eps": 1e-6})
        return (got[0] if residual else v,) + tuple(got[1 if residual else 0:]) + (() if out in EIGHT_BITS else (None,))

    def product(y, scale, w, factor, outputs):
        if not eight:
            return x.dot(y, w, (1, 1))
        f = x.binary("multiply", x.dot(y, w, (1, 1), "f32"), x.spread(scale, [0], [t, outputs]))
        return x.convert(x.binary("multiply", f, x.spread(factor, [], [t, outputs])), dt)

    h, late, caches = x.reshape(x.operator("rx.embedding", [table, tokens], [([b, n, width], dt)], {"scale": 1.0})[0], [t, width]), None, []
    for w in weights:
        factor = w.get("factor", {})
        h, y, scale = normed(late or h, h if late else None, w["norm1"], products)
        q, k, v = (x.reshape(product(y, scale, w[key], factor.get(key), heads * head_dim), [t, heads, head_dim]) for key, heads in (("q", q_heads), ("k", kv_heads), ("v", kv_heads)))
        q, *now = x.operator("rx.kv_write", [q, k, v, cos, sin, angle, position, sequence, pages] + w["caches"],
                             [([t, q_heads, head_dim], dt)] + [x.shapes[c] for c in w["caches"]], {"rotation": rotation, "layout": layout, "sections": ",".join(map(str, sections))})
        caches += now
        a = x.operator("rx.tree_attention", [x.reshape(q, [b, n, q_heads, head_dim]), now[0], now[1], pages, lengths, mask] + now[2:], [([b, n, q_heads, head_dim], dt)], {"layout": layout})[0]
        h, y, scale = normed(x.dot(x.reshape(a, [t, q_heads * head_dim]), w["o"], (1, 1)), h, w["norm2"], products)
        gate, up = (product(y, scale, w[key], factor.get(key), hidden) for key in ("gate", "up"))
        act = x.binary("multiply", gate, x.op("logistic %s : (%s)" % (gate, x.types[gate]), [t, hidden], dt))
        late = x.dot(x.binary("multiply", act, up), w["down"], (1, 1))
    y = normed(late, h, norm, dt)[1]
    logits = x.dot(y, head, (1, 1))
    one = ([t], "f32")
    out = x.operator("rx.token_logprobs", [logits, x.reshape(targets, [t])], [one, one, one, ([t, top], "f32"), ([t, top], "i32")], {"top": top})
    return x.module("verify_step", out + caches), [x.shapes["%%arg%d" % k] for k in range(len(x.args))], list(range(first_cache, first_cache + held * layers))


def tied_head_step(tokens, vocab, width, dt="f32", entropy_weight=0.0):
    """Loss and gradient of a model that is one table: rows of the tokens, logits against the whole table, the mean negative
    log probability of the targets minus `entropy_weight` times the mean entropy.  (table, ids, targets) -> (loss, the table's
    gradient): the log probabilities' gradient goes back through the product to the rows and into the table twice, as an
    operand of the product and through the lookup."""
    x = _Text()
    table, ids, targets = x.arg([vocab, width], dt), x.arg([tokens], "i32"), x.arg([tokens], "i32")
    h = x.operator("rx.embedding", [table, ids], [([tokens, width], dt)], {"scale": 1.0})[0]
    logits = x.dot(h, table, (1, 1))
    one = ([tokens], "f32")
    logprob, lse, entropy = x.operator("rx.token_logprobs", [logits, targets], [one, one, one], {"top": 0})
    weighted = x.binary("multiply", entropy, x.constant("%.9e" % entropy_weight, [tokens], "f32"))
    each = x.binary("add", logprob, weighted)
    total = x.op("reduce(%s init: %s) applies stablehlo.add across dimensions = [0] : (%s, tensor<f32>)"
                 % (each, x.constant("0.000000e+00", [], "f32"), x.types[each]), [], "f32")
    loss = x.binary("multiply", total, x.constant("%.9e" % (-1.0 / tokens), [], "f32"))
    g, e = x.constant("%.9e" % (-1.0 / tokens), [tokens], "f32"), x.constant("%.9e" % (-entropy_weight / tokens), [tokens], "f32")
    d = x.operator("rx.token_logprobs_grad", [logits, targets, lse, entropy, g, e], [([tokens, vocab], dt)])[0]
    dh = x.dot(d, table, (1, 0))
    rows = x.operator("rx.embedding_grad", [dh, ids], [([vocab, width], dt)], {"scale": 1.0})[0]
    return x.module("tied_head_step", [loss, x.binary("add", x.dot(d, h, (0, 0)), rows)])
