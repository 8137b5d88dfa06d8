"""Operators of a model that is served in 8 bits and drafts its tokens, and of the training of its norms, called as a user's
program calls them: modules with the `rx.*` operators are compiled through the framework's public entry points, and the thunks
are called on device arrays.

    norm        sum with the residual and root-mean-square norm, in the input's type or in 8 bits      rx.rms_norm
    norm_grad   its gradient by the input and by the weight                                            rx.rms_norm_grad
    write       keys and values, turned by positions of several axes, into a paged cache, in 8 bits    rx.kv_write
    move        the slots of accepted drafted tokens moved together                                    rx.kv_move
    attention   drafted tokens of a tree, or one new token, over a paged cache, also one of 8 bits     rx.tree_attention

With `own` false `run` computes the same in elementary torch operations in 32 bits, rounded once at the end.  Numbers of 8
bits are results of their own beside the scales that belong to them."""
import importlib
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "f8E4M3FN": torch.float8_e4m3fn, "i8": torch.int8, "i1": torch.bool}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "f8E4M3FN": 1, "i8": 1}
_LARGEST = {"f8E4M3FN": 448.0, "i8": 127.0}
EPS = 1e-6
SMALLEST = 2.0 ** -100      # what the scale of a row of smaller numbers is made from


def listed():
    return [
        # between two layers of a decoding step, for a product in 8 bits: a call that is all latency
        {"name": "norm_decode", "kind": "norm", "rows": 48, "width": 4096, "residual": True, "dt": "bf16", "out": "f8E4M3FN"},
        # the same for a large batch of prompts
        {"name": "norm_batch", "kind": "norm", "rows": 16384, "width": 4096, "residual": True, "dt": "bf16", "out": "f8E4M3FN"},
        # training a small model in single precision: a ragged batch, rows of no whole vectors
        {"name": "norm_grad_small", "kind": "norm_grad", "rows": 513, "width": 1001, "residual": False, "dt": "f32"},
        # one step's tokens of a large training batch
        {"name": "norm_grad_batch", "kind": "norm_grad", "rows": 16384, "width": 4096, "residual": True, "dt": "bf16"},
        # one decoding step's new tokens into a cache of 8 bits: latency again
        {"name": "write_decode", "kind": "write", "tokens": 48, "sequences": 48, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "slots": 16384, "rotary": 128, "axes": 1, "rotation": "halves", "layout": "slots", "dt": "bf16", "cache": "f8E4M3FN"},
        # prompts with images or video: positions in time, height and width, several sequences of uneven lengths
        {"name": "write_video", "kind": "write", "tokens": 8191, "sequences": 5, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "slots": 32768, "rotary": 128, "axes": 3, "rotation": "halves", "layout": "heads", "dt": "bf16", "cache": "f8E4M3FN"},
        # the branches that a served batch accepts, in 8 bits
        {"name": "move_decode", "kind": "move", "sequences": 48, "steps": 5, "drafted": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "longest": 512,
         "layout": "slots", "cache": "f8E4M3FN"},
        # long branches of a large batch, 16-bit caches, a page's slots of a head together
        {"name": "move_batch", "kind": "move", "sequences": 256, "steps": 16, "drafted": 64, "kv_heads": 8, "head_dim": 128, "page": 64, "longest": 512,
         "layout": "heads", "cache": "bf16"},
        # a single user's drafted tokens: the cache is split over the whole chip
        {"name": "tree_one", "kind": "attention", "sequences": 1, "drafted": 8, "tree": True, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "longest": 1000, "spread": "equal", "layout": "slots", "dt": "bf16", "cache": "bf16"},
        # a served batch of sequences of very different lengths, trees of 16 tokens over a cache of 8 bits
        {"name": "tree_batch", "kind": "attention", "sequences": 64, "drafted": 16, "tree": True, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "longest": 8192, "spread": "log", "layout": "slots", "dt": "bf16", "cache": "f8E4M3FN"},
        # one new token over long contexts in 8 bits: 8 sequences of 131072 positions, 2.1 GB of keys and values
        {"name": "decode_long", "kind": "attention", "sequences": 8, "drafted": 1, "tree": False, "q_heads": 64, "kv_heads": 8, "head_dim": 128, "page": 64,
         "longest": 131072, "spread": "equal", "layout": "heads", "dt": "bf16", "cache": "f8E4M3FN"},
        # wide trees, many query heads to a key head, pages of no power of two: bound by arithmetic
        {"name": "tree_wide", "kind": "attention", "sequences": 16, "drafted": 64, "tree": True, "q_heads": 64, "kv_heads": 8, "head_dim": 128, "page": 24,
         "longest": 4001, "spread": "equal", "layout": "slots", "dt": "f16", "cache": "f16"},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "write", "move", "attention", "attention", "attention"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "norm_grad"):
        case = {"kind": kind, "rows": _log(rng, 1, 16384), "width": rng.choice([64, 100, 512, 768, 1024, 1001, 2048, 4096]), "residual": rng.random() < 0.75, "dt": dt}
        if dt == "f32":
            case["rows"] = min(case["rows"], 8192)
        if kind == "norm":
            case["out"] = rng.choice([dt, "f8E4M3FN"])
        return case
    heads = {"kv_heads": rng.choice([1, 2, 4, 8, 12]), "head_dim": rng.choice([64, 80, 96, 128, 192, 256])}
    common = {"page": rng.choice([1, 16, 24, 64, 128]), "layout": rng.choice(["slots", "heads"])}
    if kind == "move":
        steps = _log(rng, 1, 16)
        return dict(heads, **common, kind=kind, sequences=_log(rng, 1, 256), steps=steps, drafted=steps + _log(rng, 1, 48), longest=512,
                    cache=rng.choice([dt, "f8E4M3FN", "i8"]))
    heads["q_heads"] = heads["kv_heads"] * rng.choice([1, 2, 4, 7, 8, 16])
    if kind == "write":
        tokens = _log(rng, 1, 8192 * 40 * 128 // (max(40, heads["q_heads"] + 2 * heads["kv_heads"]) * heads["head_dim"]))
        return dict(heads, **common, kind=kind, tokens=tokens, sequences=rng.randint(1, min(tokens, 64)), slots=32768, rotary=heads["head_dim"] // rng.choice([1, 1, 2]),
                    axes=rng.choice([1, 2, 3]), rotation=rng.choice(["halves", "pairs"]), dt=dt, cache=rng.choice([dt, "f8E4M3FN", "f8E4M3FN"]))
    case = dict(heads, **common, kind=kind, sequences=_log(rng, 1, 128), drafted=rng.choice([1, 1, 4, 7, 16, 33, 64]), tree=rng.random() < 0.75, longest=0,
                spread=rng.choice(["equal", "log", "log"]), dt=dt, cache=rng.choice([dt, "f8E4M3FN", "i8"]))
    b, rows = case["sequences"], case["sequences"] * case["drafted"] * case["q_heads"]
    token = 2.0 * case["kv_heads"] * case["head_dim"] * _SIZE[case["cache"]] * b   # bytes of one position of all sequences
    # the plain form pads to the longest and works in 32 bits; both bounded by what the largest listed cases take
    case["longest"] = _log(rng, 1, int(max(1, min(131072, 1.0e9 / token, 4.0e8 / rows, (3.0e11 if dt != "f32" else 1.0e11) / (4.0 * rows * case["head_dim"])))))
    return case


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------
def _lengths(case):
    """The sequences' positions before the drafted tokens, longest first; they depend on the case alone, and the seed decides
    whose is which.  In a large batch some places are not taken (-1)."""
    b, longest = case["sequences"], case["longest"]
    if case["kind"] == "move" or case["spread"] == "equal":
        return [longest] * b
    return [-1 if b >= 16 and k >= b - b // 16 else int(round(longest ** (1.0 - k / max(1, b - 1)))) - (k > 0) for k in range(b)]


def _cache_shape(case, pages):
    h, d, s = case["kv_heads"], case["head_dim"], case["page"]
    return (pages, s, h, d) if case["layout"] == "slots" else (pages, h, s, d)


def _needed(case):
    """Pages of every sequence, of those of _lengths."""
    return [-(-(n + case["drafted"]) // case["page"]) if n >= 0 else 0 for n in _lengths(case)]


def _pages(case):
    """(pages of the cache, columns of the page table)"""
    if case["kind"] == "write":
        return -(-case["slots"] // case["page"]) + case["sequences"], -(-case["slots"] // case["page"])
    return sum(_needed(case)) + 3, max(1, max(_needed(case)))


def _sections(case):
    """Pairs of the rotated dimensions that follow each axis: the first takes what is left."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    return [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)


def _axis_of(case, device):
    return torch.repeat_interleave(torch.arange(case["axes"], device=device), torch.tensor(_sections(case), device=device))


def _quantized(x, dt):
    """(numbers of 8 bits, scales of the last dimension's rows) of values in 32 bits."""
    largest = torch.full((), _LARGEST[dt], device=x.device)
    scale = x.abs().amax(-1).clamp(min=SMALLEST) / largest
    y = x / scale[..., None]
    return (y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn) if dt == "f8E4M3FN" else y.round().to(torch.int8)), scale


def _inputs(case, seed):
    gen = torch.Generator()
    gen.manual_seed(int(seed))
    dev = torch.Generator(device="cuda")
    dev.manual_seed(int(seed))
    kind = case["kind"]

    def normal(*shape, dt=None):
        dt = _TORCH[dt or case["dt"]]
        return torch.randn(shape, generator=dev, device="cuda", dtype=dt)

    def cache(pages):
        """Keys and values that the cache holds, with their scales in 8 bits."""
        shape, dt = _cache_shape(case, pages), case["cache"]
        if dt not in _LARGEST:
            return {"k_cache": normal(*shape, dt=dt), "v_cache": normal(*shape, dt=dt)}
        out = {}
        for name in ("k", "v"):
            codes = torch.empty(shape, device="cuda", dtype=_TORCH[dt])
            scales = torch.empty((pages, case["kv_heads"], case["page"]), device="cuda")     # a head's scales of a page lie together
            step = max(1, (1 << 28) // max(1, int(np.prod(shape[1:]))))
            for lo in range(0, pages, step):                 # not all in 32 bits at once
                x = torch.randn((min(step, pages - lo),) + shape[1:], generator=dev, device="cuda")
                codes[lo:lo + step], s = _quantized(x, dt)
                scales[lo:lo + step] = s.transpose(1, 2) if case["layout"] == "slots" else s
            out[name + "_cache"], out[name + "_scale"] = codes, scales
        return {k: out[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}

    if kind == "norm":
        out = {"x": normal(case["rows"], case["width"])}
        if case["residual"]:
            out["residual"] = normal(case["rows"], case["width"]) * 4.0
        out["weight"] = (1.0 + 0.2 * torch.randn(case["width"], generator=gen)).to(_TORCH[case["dt"]]).cuda()
        return out
    if kind == "norm_grad":
        out = {"h": normal(case["rows"], case["width"]) * 4.0, "weight": (1.0 + 0.2 * torch.randn(case["width"], generator=gen)).to(_TORCH[case["dt"]]).cuda(),
               "dy": normal(case["rows"], case["width"])}
        if case["residual"]:
            out["dh"] = normal(case["rows"], case["width"])
        return out
    pages, cols = _pages(case)
    order = torch.randperm(pages, generator=gen).int()
    if kind == "write":
        t, b, r = case["tokens"], case["sequences"], case["rotary"]
        # tokens of the sequences one after the other; each sequence already holds a few
        cut = sorted(torch.randperm(t - 1, generator=gen)[:b - 1].tolist()) if b > 1 else []
        ends = [c + 1 for c in cut] + [t]
        begins = [0] + ends[:-1]
        room = (case["slots"] - t) // b
        position, sequence, need = [], [], []
        for s, (lo, hi) in enumerate(zip(begins, ends)):
            held = int(torch.randint(0, room + 1, (1,), generator=gen))
            position += range(held, held + hi - lo)
            sequence += [s] * (hi - lo)
            need.append(-(-(held + hi - lo) // case["page"]))
        table = torch.full((b, cols), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        position = torch.tensor(position, dtype=torch.int32)
        # the first axis follows the position (time), the others are places within an image of 32 columns
        axes = [position] + [(position if a == 1 else position // 32) % 32 for a in range(1, case["axes"])]
        angle = torch.stack(axes).clone()
        if t >= 64:
            position[torch.randperm(t, generator=gen)[:t // 64]] = -1       # padding
        turn = torch.arange(case["slots"], device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r))[None, :]
        return {"q": normal(t, case["q_heads"], case["head_dim"]), "k": normal(t, case["kv_heads"], case["head_dim"]),
                "v": normal(t, case["kv_heads"], case["head_dim"]), "cos": turn.cos().float(), "sin": turn.sin().float(), "angle": angle.cuda(),
                "position": position.cuda(), "sequence": torch.tensor(sequence, dtype=torch.int32).cuda(), "pages": table.cuda(), **cache(pages)}
    b = case["sequences"]
    mix = torch.randperm(b, generator=gen)
    lengths, need = torch.tensor(_lengths(case), dtype=torch.int32)[mix], torch.tensor(_needed(case))[mix]
    table = torch.full((b, cols), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need.tolist()):
        table[s, :n] = order[at:at + n]
        at += n
    if kind == "move":
        # a branch: the first drafted token, then ever later ones that lie behind all places that are moved to
        steps, drafted = case["steps"], case["drafted"]
        path = torch.full((b, steps), -1, dtype=torch.int32)
        taken = torch.randint(1, steps + 1, (b,), generator=gen).tolist()
        for s, n in enumerate(taken):
            n = min(n, drafted - steps + 1)
            path[s, 0] = 0
            path[s, 1:n] = steps + torch.randperm(drafted - steps, generator=gen)[:n - 1].sort().values.int()
        return {"lengths": lengths.cuda(), "path": path.cuda(), "pages": table.cuda(), **cache(pages)}
    n = case["drafted"]
    out = {"q": normal(b, n, case["q_heads"], case["head_dim"])}
    stored = cache(pages)
    out.update(k_cache=stored["k_cache"], v_cache=stored["v_cache"], pages=table.cuda(), lengths=lengths.cuda())
    if case["tree"]:
        # a token sees itself and its ancestors; trees of fewer tokens leave the last rows empty
        size = torch.randint(max(1, n // 2), n + 1, (b,), generator=gen).numpy()
        parent = np.floor(torch.rand((b, n), generator=gen).numpy() * (np.arange(n) + 1)[None, :]).astype(np.int64) - 1
        mask = np.zeros((b, n, n), dtype=bool)
        for i in range(n):
            mask[:, i] = np.where((parent[:, i] >= 0)[:, None], mask[np.arange(b), np.maximum(parent[:, i], 0)], False)
            mask[:, i, i] = True
        mask &= (np.arange(n)[None, :] < size[:, None])[:, :, None]
        out["mask"] = torch.from_numpy(mask).cuda()
    if case["cache"] in _LARGEST:
        out.update(k_scale=stored["k_scale"], v_scale=stored["v_scale"])
    return out


# ----------------------------------------------------------------------------
# the framework's calls
# ----------------------------------------------------------------------------
def _package():
    if "reactant_jl_amd" not in sys.modules:
        d = os.path.abspath("reactant.jl_amd")
        spec = importlib.util.spec_from_file_location("reactant_jl_amd", os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["reactant_jl_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["reactant_jl_amd"]


def _program(case):
    P = importlib.import_module("reactant_jl_amd.lm_programs")
    kind = case["kind"]
    if kind == "norm":
        return P.rms_norm(case["rows"], case["width"], dt=case["dt"], out=case["out"], eps=EPS, residual=case["residual"])
    if kind == "norm_grad":
        return P.rms_norm_grad(case["rows"], case["width"], dt=case["dt"], eps=EPS, residual=case["residual"])
    pages, cols = _pages(case)
    if kind == "write":
        return P.kv_write(case["tokens"], case["sequences"], case["q_heads"], case["kv_heads"], case["head_dim"], pages, case["page"], cols, case["slots"], dt=case["dt"],
                          cache=case["cache"], sections=_sections(case), rotation=case["rotation"], layout=case["layout"])
    if kind == "move":
        return P.kv_move(case["sequences"], case["steps"], case["kv_heads"], case["head_dim"], pages, case["page"], cols, cache=case["cache"], layout=case["layout"])
    return P.tree_attention(case["sequences"], case["drafted"], case["q_heads"], case["kv_heads"], case["head_dim"], pages, case["page"], cols, dt=case["dt"],
                            cache=case["cache"], mask=case["tree"], layout=case["layout"])


class _Bytes:
    """A device array's memory as torch takes it; torch keeps this object, and with it the array, while its view lives."""

    TYPESTR = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4", "f8E4M3FN": "|u1", "i8": "|i1", "i1": "|u1"}

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = {"shape": array.shape[::-1], "typestr": self.TYPESTR[array.dtype], "version": 2,
                                         "data": (array.data.buffer.unsafe_pointer(), False)}


def _view(array):
    t = torch.as_tensor(_Bytes(array), device="cuda")
    return t.view(_TORCH[array.dtype]) if array.dtype in ("bf16", "f8E4M3FN", "i1") else t


_compiled = {}


def prepare(case, seed):
    inputs = _inputs(case, seed)
    if not own:
        return {"case": case, "inputs": inputs}
    rx = _package()
    client = rx.set_default_backend("gpu")
    text = _program(case)
    if text not in _compiled:
        _compiled[text] = rx.compile(text)
    client.default_device().synchronize()         # a recycled block may still be in use on the framework's stream
    names = {v: k for k, v in _TORCH.items()}
    arrays = []
    for key in list(inputs):
        t = inputs.pop(key)
        dt = names[t.dtype]
        array = rx.ConcreteRArray(rx.AsyncBuffer(rx.Buffer.uninitialized(client, tuple(t.shape), dt)), tuple(t.shape)[::-1], dt)
        _view(array).copy_(t)
        arrays.append(array)
    torch.cuda.synchronize()                      # nor does that stream wait for torch's
    return {"case": case, "thunk": _compiled[text], "args": arrays}


# ----------------------------------------------------------------------------
# the plain forms
# ----------------------------------------------------------------------------
def _plain_rotate(x, cos, sin, rotation):
    r = 2 * cos.shape[-1]
    x, c, s = x.float(), cos[:, None, :], sin[:, None, :]
    if rotation == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _put(cache, page, slot, new, layout):
    if layout == "slots":
        cache[page, slot] = new
    else:
        cache[page, :, slot] = new


def _raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain(case, x):
    kind = case["kind"]
    if kind == "norm":
        h = x["x"].float() + x["residual"].float() if case["residual"] else x["x"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * x["weight"].float()
        first = [h.to(_TORCH[case["dt"]])] if case["residual"] else []
        return first + (list(_quantized(y, case["out"])) if case["out"] in _LARGEST else [y.to(_TORCH[case["dt"]])])
    if kind == "norm_grad":
        h, dy = x["h"].float(), x["dy"].float()
        g = dy * x["weight"].float()
        r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        dx = r * (g - h * (r * r * (g * h).mean(-1, keepdim=True)))
        if case["residual"]:
            dx = dx + x["dh"].float()
        return [dx.to(_TORCH[case["dt"]]), (dy * h * r).sum(0)]
    if kind == "write":
        position = x["position"].long()
        known = position >= 0
        at = torch.where(known, position, 0)
        column = torch.arange(case["rotary"] // 2, device=at.device)
        rows = x["angle"].long()[_axis_of(case, at.device)].t()                # [token, pair]
        cos, sin = x["cos"][rows, column], x["sin"][rows, column]
        q = torch.where(known[:, None, None], _plain_rotate(x["q"], cos, sin, case["rotation"]), 0.0).to(_TORCH[case["dt"]])
        keep = known.nonzero()[:, 0]
        page = x["pages"][x["sequence"].long(), at // case["page"]].long()[keep]
        slot = (at % case["page"])[keep]
        for name, new in (("k", _plain_rotate(x["k"], cos, sin, case["rotation"])), ("v", x["v"].float())):
            if case["cache"] in _LARGEST:
                new, scale = _quantized(new, case["cache"])
                _put(x[name + "_scale"], page, slot, scale[keep], "heads")
            else:
                new = new.to(_TORCH[case["cache"]])
            _put(_raw(x[name + "_cache"]), page, slot, _raw(new)[keep], case["layout"])
        return [q, x["k_cache"], x["v_cache"]] + ([x["k_scale"], x["v_scale"]] if case["cache"] in _LARGEST else [])
    caches = [x[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale") if k in x]
    if kind == "move":
        path, base = x["path"].long(), x["lengths"].long()[:, None]
        b, i = (path >= 0).nonzero(as_tuple=True)
        to, source = (base + torch.arange(case["steps"], device=path.device))[b, i], (base + path)[b, i]
        pages = x["pages"].long()
        to, source = ((pages[b, t // case["page"]], t % case["page"]) for t in (to, source))
        for cache, layout in zip(map(_raw, caches), [case["layout"]] * 2 + ["heads"] * 2):
            _put(cache, *to, cache[source] if layout == "slots" else cache[source[0], :, source[1]], layout)
        return caches
    b, n, hq, d = x["q"].shape
    hk, lengths = case["kv_heads"], x["lengths"].long()
    pages = torch.clamp(x["pages"].long(), min=0)

    def gathered(name):
        t = _raw(x[name + "_cache"])[pages].view(x[name + "_cache"].dtype).float()     # [sequence, page, ..]
        if case["layout"] == "heads":
            t = t.transpose(2, 3)
        if name + "_scale" in x:
            t = t * x[name + "_scale"][pages].transpose(2, 3)[..., None]
        return t.reshape(b, -1, hk, d).permute(0, 2, 1, 3).contiguous()       # [sequence, head, position, dim]
    q = x["q"].float().reshape(b, n, hk, hq // hk, d).transpose(1, 2).reshape(b, hk, -1, d)
    s = torch.matmul(q, gathered("k").transpose(2, 3).contiguous()) / math.sqrt(d)
    late = torch.arange(s.shape[-1], device=s.device)[None, :] - lengths[:, None]     # the drafted token that a position holds
    mask = x["mask"] if case["tree"] else torch.ones((n, n), device=s.device, dtype=torch.bool).tril().expand(b, n, n)
    there = torch.where((late < 0)[:, None], True, mask.gather(2, late.clamp(0, n - 1)[:, None].expand(b, n, -1)) & (late < n)[:, None])
    there &= (lengths >= 0)[:, None, None]
    s = torch.where(there[:, None, :, None, :], s.reshape(b, hk, n, hq // hk, -1), -math.inf).reshape(s.shape)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, gathered("v")) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, hk, n, hq // hk, d).transpose(1, 2).reshape(b, n, hq, d).to(_TORCH[case["dt"]])


def run(state):
    if not own:
        return _plain(state["case"], state["inputs"])
    args, case = state["args"], state["case"]
    if case["kind"] in ("write", "move"):
        caches = 4 if case["cache"] in _LARGEST else 2
        out = state["thunk"](*args, donated=[False] * (len(args) - caches) + [True] * caches)
        args[-caches:] = out[-caches:]            # the caches live on in the results
    else:
        out = state["thunk"](*args)
    return [_view(o) for o in out] if isinstance(out, tuple) else _view(out)


# ----------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = float(case["rows"]) * case["width"], _SIZE[case["dt"]]
        return {"bytes": n * (e * (3 if case["residual"] else 1) + _SIZE[case["out"]]) + e * case["width"], "flops": 6.0 * n}
    if kind == "norm_grad":
        n, e = float(case["rows"]) * case["width"], _SIZE[case["dt"]]
        return {"bytes": n * e * (4 if case["residual"] else 3) + (e + 4.0) * case["width"], "flops": 11.0 * n}
    slot = 2.0 * case["kv_heads"] * (case["head_dim"] * _SIZE[case["cache"]] + (4 if case["cache"] in _LARGEST else 0))      # bytes of a position in the caches
    if kind == "move":
        moved = case["sequences"] * (case["steps"] - 1) / 2.0
        return {"bytes": 2.0 * slot * moved + 4.0 * case["sequences"] * (case["steps"] + 1), "flops": 0.0}
    e, d = _SIZE[case["dt"]], case["head_dim"]
    if kind == "write":
        t = float(case["tokens"])
        return {"bytes": e * t * d * 2 * (case["q_heads"] + case["kv_heads"]) + slot * t + 4.0 * t * (case["rotary"] + 2 + case["axes"]),
                "flops": 3.0 * t * (case["q_heads"] + case["kv_heads"]) * case["rotary"]}
    new, taken = case["drafted"], [n for n in _lengths(case) if n >= 0]
    n = float(sum(taken) + new * len(taken))
    return {"bytes": slot * n + 2.0 * e * case["sequences"] * new * case["q_heads"] * d + 4.0 * (n / case["page"] + case["sequences"]),
            "flops": 4.0 * n * new * case["q_heads"] * d}


# ----------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------
def _codes(x, dt):
    scale = torch.clamp(x.abs().amax(-1), min=SMALLEST) / _LARGEST[dt]
    y = x / scale[..., None]
    return (y.float().clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double() if dt == "f8E4M3FN" else None), scale


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h, w = x["x"].double(), x["weight"].double()
        if case["residual"]:
            h += x["residual"].double()
        y = h / torch.sqrt((h ** 2).sum(-1) / case["width"] + EPS)[:, None] * w
        return ([h] if case["residual"] else []) + (list(_codes(y, case["out"])) if case["out"] in _LARGEST else [y])
    if kind == "norm_grad":
        parts, total = [], torch.zeros(case["width"], device="cuda", dtype=torch.float64)
        for lo in range(0, case["rows"], 2048):
            h, dy = (x[k][lo:lo + 2048].double() for k in ("h", "dy"))
            rms = torch.sqrt((h ** 2).sum(-1, keepdim=True) / case["width"] + EPS)
            unit = h / rms                                                     # y = unit * weight
            back = dy * x["weight"].double()
            dx = (back - unit * (back * unit).sum(-1, keepdim=True) / case["width"]) / rms
            parts.append(dx + x["dh"][lo:lo + 2048].double() if case["residual"] else dx)
            total += (dy * unit).sum(0)
        return [torch.cat(parts), total]
    if kind == "write":
        position, half = x["position"].long(), case["rotary"] // 2
        there = position >= 0
        rows = torch.cat([x["angle"][a].long()[:, None].expand(-1, m) for a, m in enumerate(_sections(case))], 1)
        turn = torch.complex(x["cos"].double().gather(0, rows), x["sin"].double().gather(0, rows))[:, None, :]   # rotation = product with a unit number
        q, k = x["q"].double(), x["k"].double()
        for t in (q, k):
            if case["rotation"] == "halves":
                z = torch.complex(t[..., :half], t[..., half:2 * half]) * turn
                t[..., :half], t[..., half:2 * half] = z.real, z.imag
            else:
                z = torch.complex(t[..., 0:2 * half:2], t[..., 1:2 * half:2]) * turn
                t[..., 0:2 * half:2], t[..., 1:2 * half:2] = z.real, z.imag
        q[~there] = 0.0
        pages = x["pages"][x["sequence"].long()[there], position[there] // case["page"]].long()
        slots = position[there] % case["page"]
        caches, scales = [], []
        for name, new in (("k", k), ("v", x["v"].double())):
            held = x[name + "_cache"].double()
            if case["cache"] in _LARGEST:
                new, scale = _codes(new, case["cache"])
                held_scale = x[name + "_scale"].double()
                held_scale.transpose(1, 2).index_put_((pages, slots), scale[there])
                scales.append(held_scale)
            (held if case["layout"] == "slots" else held.transpose(1, 2)).index_put_((pages, slots), new[there])
            caches.append(held)
        return [q] + caches + scales
    if kind == "move":
        out = []
        for key in ("k_cache", "v_cache", "k_scale", "v_scale"):
            if key not in x:
                continue
            cache = x[key].double()
            rows = cache if case["layout"] == "slots" and key.endswith("cache") else cache.transpose(1, 2)
            held = rows.clone()
            b, i = (x["path"] >= 0).nonzero(as_tuple=True)
            n, pages = x["lengths"].long()[b], x["pages"].long()
            to, source = n + i, n + x["path"].long()[b, i]
            rows.index_put_((pages[b, to // case["page"]], to % case["page"]), held[pages[b, source // case["page"]], source % case["page"]])
            out.append(cache if x[key].dtype != torch.int8 else None)
        return out
    hk, g, d, n = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"], case["drafted"]
    out = torch.zeros(x["q"].shape, device="cuda", dtype=torch.float64)
    for b, length in enumerate(x["lengths"].tolist()):
        if length < 0:
            continue
        pages = x["pages"][b, :-(-(length + n) // case["page"])].long()
        sees = torch.ones((n, length + n), device="cuda", dtype=torch.bool)
        sees[:, length:] = x["mask"][b] if case["tree"] else torch.arange(n, device="cuda")[:, None] >= torch.arange(n, device="cuda")[None, :]
        some = sees.any(-1)
        if not bool(some.any()):
            continue
        for h in range(hk):
            k, v = (((_raw(c)[pages, :, h] if case["layout"] == "slots" else _raw(c)[pages, h]).view(c.dtype)).reshape(-1, d)[:length + n].double() for c in (x["k_cache"], x["v_cache"]))
            if "k_scale" in x:
                k, v = (t * s[pages, h].reshape(-1, 1)[:length + n].double() for t, s in ((k, x["k_scale"]), (v, x["v_scale"])))
            q = x["q"][b, some, h * g:(h + 1) * g].double()                    # [token, head, dim]
            s = (q.reshape(-1, d) @ k.t() / math.sqrt(d)).reshape(q.shape[0], g, -1)
            w = torch.softmax(s.masked_fill(~sees[some][:, None], -math.inf), -1)
            out[b, some, h * g:(h + 1) * g] = (w.reshape(-1, length + n) @ v).reshape(q.shape)
    return out
