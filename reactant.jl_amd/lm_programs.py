"""Module text of the language-model operators: `stablehlo.custom_call` of the backend's `rx.` targets, and programs that
use them together.  Like programs.py this stands in for the tracing front end; a traced program holds the same calls
(`MLIR.Dialects.stablehlo.custom_call` with `call_target_name` and a `backend_config` dictionary, reference
src/mlir/Dialects/StableHLO.jl).

Each writer names its shapes in the module's row-major order and returns text for `compile`; what the targets compute is
stated in csrc/rx_lm.h.  Arguments come in the order of the operands.  Cache arguments are marked with the result that may
take them over: a call with them donated updates the caches in place, one without copies them first."""


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

    def constant(self, literal, shape, dt):
        self.n += 1
        name = "%%c%d" % self.n
        self.types[name], self.shapes[name] = tt(shape, dt), (list(shape), dt)
        self.lines.append("    %s = stablehlo.constant dense<%s> : %s\n" % (name, literal, tt(shape, dt)))
        return name

    def iota(self, n):
        self.n += 1
        name = "%%v%d" % self.n
        self.types[name], self.shapes[name] = tt([n], "i32"), ([n], "i32")
        self.lines.append("    %s = stablehlo.iota dim = 0 : %s\n" % (name, tt([n], "i32")))
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
