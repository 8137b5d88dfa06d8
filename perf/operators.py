"""The operators of language models whose time counts, called as a user's program calls them: modules with the
`rx.*` operators are compiled through the framework's public entry points, and the thunks are called on device arrays.

    embedding     rows of a table by token, scaled                               rx.embedding
    embed_grad    its gradient, every row's tokens summed in their order         rx.embedding_grad
    append        rotated keys and values into a paged cache                     rx.kv_append
    attention     one new token per sequence over a paged cache                  rx.paged_attention
    logprobs      log probabilities of tokens, entropy, top alternatives         rx.token_logprobs
    logprob_grad  gradient of log probability and entropy by the logits          rx.token_logprobs_grad

With `own` false `run` computes the same in elementary torch operations in 32 bits, rounded once at the end."""
import importlib
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one step's tokens of a large training batch: rows of a model's table
        {"name": "embedding_batch", "kind": "embedding", "tokens": 16384, "rows": 32000, "width": 4096, "dt": "bf16", "scale": 1.0},
        # gradient of a small model's table for a short, ragged batch: launches count
        {"name": "embed_grad_small", "kind": "embed_grad", "tokens": 513, "rows": 10007, "width": 1024, "dt": "f32", "out": "f32", "scale": 32.0},
        # gradient of a large table in f32 from 16-bit activations, with frequent tokens as text has them
        {"name": "embed_grad_large", "kind": "embed_grad", "tokens": 16384, "rows": 65536, "width": 4096, "dt": "bf16", "out": "f32", "scale": 1.0},
        # one decoding step's new tokens: a call that is all latency
        {"name": "append_decode", "kind": "append", "tokens": 48, "sequences": 48, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "slots": 16384, "rotary": 128, "rotation": "halves", "layout": "slots", "dt": "bf16"},
        # prompts of several sequences that arrive together, of uneven lengths, pairs rotated over part of a head
        {"name": "append_prompts", "kind": "append", "tokens": 8191, "sequences": 5, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "slots": 32768, "rotary": 64, "rotation": "pairs", "layout": "heads", "dt": "f16"},
        # a single user's next token: the cache is split over the whole chip
        {"name": "attention_one", "kind": "attention", "sequences": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "longest": 1000,
         "spread": "equal", "layout": "slots", "dt": "bf16"},
        # a served batch of sequences of very different lengths
        {"name": "attention_batch", "kind": "attention", "sequences": 64, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "longest": 8192,
         "spread": "log", "layout": "slots", "dt": "bf16"},
        # long contexts: 8 sequences of 131072 tokens, 4.3 GB of keys and values
        {"name": "attention_long", "kind": "attention", "sequences": 8, "q_heads": 64, "kv_heads": 8, "head_dim": 128, "page": 64, "longest": 131072,
         "spread": "equal", "layout": "heads", "dt": "bf16"},
        # single precision, a key head for every query head, a head of an uneven width, pages of no power of two
        {"name": "attention_f32", "kind": "attention", "sequences": 7, "q_heads": 12, "kv_heads": 12, "head_dim": 80, "page": 24, "longest": 4001,
         "spread": "log", "layout": "slots", "dt": "f32"},
        # the sampled tokens' log probabilities of a decoding batch, with alternatives
        {"name": "logprobs_decode", "kind": "logprobs", "tokens": 32, "vocab": 32000, "top": 5, "dt": "bf16"},
        # scoring a long text
        {"name": "logprobs_score", "kind": "logprobs", "tokens": 4096, "vocab": 131072, "top": 20, "dt": "bf16"},
        # the loss's gradient, a vocabulary of no whole vectors
        {"name": "logprob_grad", "kind": "logprob_grad", "tokens": 4096, "vocab": 50021, "dt": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embedding", "embed_grad", "append", "attention", "attention", "logprobs", "logprob_grad"])
    dt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("embedding", "embed_grad"):
        case = {"kind": kind, "tokens": _log(rng, 1, 16384), "rows": _log(rng, 256, 65536), "width": rng.choice([64, 100, 512, 768, 1024, 1001, 2048, 4096]),
                "dt": dt, "scale": rng.choice([1.0, 32.0])}
        if kind == "embed_grad":
            case["out"] = rng.choice([dt, "f32"])
        return case
    heads = {"q_heads": 0, "kv_heads": rng.choice([1, 2, 4, 8, 12]), "head_dim": rng.choice([64, 80, 96, 128, 192, 256])}
    heads["q_heads"] = heads["kv_heads"] * rng.choice([1, 2, 4, 7, 8, 16])
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        return dict(heads, kind=kind, tokens=tokens, sequences=rng.randint(1, min(tokens, 64)), page=rng.choice([1, 16, 24, 64, 128]),
                    slots=32768, rotary=heads["head_dim"] // rng.choice([1, 1, 2]), rotation=rng.choice(["halves", "pairs"]), layout=rng.choice(["slots", "heads"]), dt=dt)
    if kind == "attention":
        case = dict(heads, kind=kind, sequences=_log(rng, 1, 128), page=rng.choice([1, 16, 24, 64, 128]), longest=0,
                    spread=rng.choice(["equal", "log", "log"]), layout=rng.choice(["slots", "heads"]), dt=dt)
        token = 2.0 * case["kv_heads"] * case["head_dim"] * _SIZE[dt] * case["sequences"]   # bytes of one position of all sequences
        # the plain form pads to the longest and works in 32 bits: both bounded by the largest listed case's
        case["longest"] = _log(rng, 1, int(max(1, min(131072, 1.0e9 / token, 2.0e9 / (case["sequences"] * case["q_heads"] * 4)))))
        return case
    vocab = rng.choice([1000, 10007, 32000, 50021, 65536, 131072])
    tokens = _log(rng, 1, 4096)
    if tokens * vocab > 1 << 28:
        tokens = (1 << 28) // vocab
    case = {"kind": kind, "tokens": tokens, "vocab": vocab, "dt": dt}
    if kind == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20])
    return case


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------
def _lengths(case):
    """The sequences' lengths, longest first; they depend on the case alone, and the seed decides whose is which."""
    b, longest = case["sequences"], case["longest"]
    if case["spread"] == "equal":
        return [longest] * b
    return [max(1, int(round(longest ** (1.0 - k / max(1, b))))) for k in range(b)]


def _ids(case, gen):
    """Tokens with frequencies that fall with their rank, as text has them; a few are padding (-1)."""
    n, rows = case["tokens"], case["rows"]
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    rank = torch.clamp((rows ** u).long() - 1, 0, rows - 1)
    stride = next(p for p in (7919, 7907, 7901) if rows % p)        # prime to the number of rows: ranks scattered over the table
    shift = int(torch.randint(0, rows, (1,), generator=gen))
    ids = ((rank * stride + shift) % rows)[torch.randperm(n, generator=gen)].int()
    if n >= 64:
        ids[torch.randperm(n, generator=gen)[:n // 64]] = -1
    return ids.cuda()


def _distinct(case):
    n, rows = case["tokens"], case["rows"]
    u = (np.arange(n) + 0.5) / n
    return len(np.unique(np.clip((rows ** u).astype(np.int64) - 1, 0, rows - 1)))


def _cache_shape(case, pages):
    h, d, s = case["kv_heads"], case["head_dim"], case["page"]
    return (pages, s, h, d) if case["layout"] == "slots" else (pages, h, s, d)


def _pages(case):
    """(pages of the cache, columns of the page table)"""
    if case["kind"] == "append":
        return -(-case["slots"] // case["page"]) + case["sequences"], -(-case["slots"] // case["page"])
    need = [-(-n // case["page"]) for n in _lengths(case)]
    return sum(need) + 3, max(need)


def _inputs(case, seed):
    gen = torch.Generator()
    gen.manual_seed(int(seed))
    dev = torch.Generator(device="cuda")
    dev.manual_seed(int(seed))
    kind, dt = case["kind"], _TORCH[case["dt"]]

    def normal(*shape):
        return torch.randn(shape, generator=dev, device="cuda", dtype=torch.float32 if dt == torch.float32 else dt)

    if kind == "embedding":
        return {"table": normal(case["rows"], case["width"]), "ids": _ids(case, gen)}
    if kind == "embed_grad":
        return {"dy": normal(case["tokens"], case["width"]), "ids": _ids(case, gen)}
    if kind == "append":
        t, b, r = case["tokens"], case["sequences"], case["rotary"]
        pages, cols = _pages(case)
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
        order = torch.randperm(pages, generator=gen).int()
        table = torch.full((b, cols), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        position = torch.tensor(position, dtype=torch.int32)
        if t >= 64:
            position[torch.randperm(t, generator=gen)[:t // 64]] = -1       # padding
        angle = torch.arange(case["slots"], device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r))[None, :]
        shape = _cache_shape(case, pages)
        return {"q": normal(t, case["q_heads"], case["head_dim"]), "k": normal(t, case["kv_heads"], case["head_dim"]),
                "v": normal(t, case["kv_heads"], case["head_dim"]), "cos": angle.cos().float(), "sin": angle.sin().float(),
                "position": position.cuda(), "sequence": torch.tensor(sequence, dtype=torch.int32).cuda(), "pages": table.cuda(),
                "k_cache": normal(*shape), "v_cache": normal(*shape)}
    if kind == "attention":
        pages, cols = _pages(case)
        lengths = torch.tensor(_lengths(case), dtype=torch.int32)[torch.randperm(case["sequences"], generator=gen)]
        order = torch.randperm(pages, generator=gen).int()
        table = torch.full((case["sequences"], cols), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(lengths.tolist()):
            n = -(-n // case["page"])
            table[s, :n] = order[at:at + n]
            at += n
        shape = _cache_shape(case, pages)
        return {"q": normal(case["sequences"], case["q_heads"], case["head_dim"]), "k_cache": normal(*shape), "v_cache": normal(*shape),
                "pages": table.cuda(), "lengths": lengths.cuda()}
    n, v = case["tokens"], case["vocab"]
    logits = normal(n, v) * 2.5
    target = torch.randint(0, v, (n,), generator=gen).int()
    logits[:, torch.randperm(v, generator=gen)[:v // 64].cuda()] = -math.inf      # tokens that may not be chosen
    if n >= 16:
        target[torch.randperm(n, generator=gen)[:n // 16]] = -1                   # positions that do not count
    out = {"logits": logits, "target": target.cuda()}
    if kind == "logprob_grad":                                                    # what the forward pass kept
        lse, entropy = (torch.empty(n, device="cuda", dtype=torch.float32) for _ in range(2))
        for lo in range(0, n, 1024):
            x = logits[lo:lo + 1024].double()
            z = torch.logsumexp(x, -1)
            p = torch.exp(x - z[:, None])
            lse[lo:lo + 1024] = z.float()
            entropy[lo:lo + 1024] = (z - torch.where(p > 0, p * x, 0.0).sum(-1)).float()
        out.update(lse=lse, entropy=entropy, d_logprob=torch.randn(n, generator=gen).cuda() - 1.0, d_entropy=0.01 * torch.rand(n, generator=gen).cuda())
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
    kind, dt = case["kind"], case["dt"]
    if kind == "embedding":
        return P.embedding(case["tokens"], case["rows"], case["width"], dt=dt, scale=case["scale"])
    if kind == "embed_grad":
        return P.embedding_grad(case["tokens"], case["rows"], case["width"], dt=dt, out=case["out"], scale=case["scale"])
    if kind == "append":
        pages, cols = _pages(case)
        return P.kv_append(case["tokens"], case["sequences"], case["q_heads"], case["kv_heads"], case["head_dim"], pages, case["page"], cols,
                           case["slots"], dt=dt, rotary_dim=case["rotary"], rotation=case["rotation"], layout=case["layout"])
    if kind == "attention":
        pages, cols = _pages(case)
        return P.paged_attention(case["sequences"], case["q_heads"], case["kv_heads"], case["head_dim"], pages, case["page"], cols, dt=dt, layout=case["layout"])
    if kind == "logprobs":
        return P.token_logprobs(case["tokens"], case["vocab"], top=case["top"], dt=dt)
    return P.token_logprobs_grad(case["tokens"], case["vocab"], dt=dt)


class _Bytes:
    """A device array's memory as torch takes it; torch keeps this object, and with it the array, while its view lives."""

    TYPESTR = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4"}

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = {"shape": array.shape[::-1], "typestr": self.TYPESTR[array.dtype], "version": 2,
                                         "data": (array.data.buffer.unsafe_pointer(), False)}


def _view(array):
    t = torch.as_tensor(_Bytes(array), device="cuda")
    return t.view(torch.bfloat16) if array.dtype == "bf16" else t


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


def _plain(case, x):
    kind, dt = case["kind"], _TORCH[case["dt"]]
    if kind == "embedding":
        ids = x["ids"].long()
        known = (ids >= 0) & (ids < case["rows"])
        return torch.where(known[:, None], x["table"][torch.where(known, ids, 0)].float() * case["scale"], 0.0).to(dt)
    if kind == "embed_grad":
        ids = x["ids"].long()
        known = (ids >= 0) & (ids < case["rows"])
        dy = torch.where(known[:, None], x["dy"].float() * case["scale"], 0.0)
        out = torch.zeros((case["rows"], case["width"]), device=dy.device, dtype=torch.float32)
        return out.index_add_(0, torch.where(known, ids, 0), dy).to(_TORCH[case["out"]])
    if kind == "append":
        position = x["position"].long()
        known = position >= 0
        at = torch.where(known, position, 0)
        cos, sin = x["cos"][at], x["sin"][at]
        q = torch.where(known[:, None, None], _plain_rotate(x["q"], cos, sin, case["rotation"]), 0.0).to(dt)
        k = _plain_rotate(x["k"], cos, sin, case["rotation"]).to(dt)
        keep = known.nonzero()[:, 0]
        page = x["pages"][x["sequence"].long(), at // case["page"]].long()[keep]
        slot = (at % case["page"])[keep]
        for cache, new in ((x["k_cache"], k), (x["v_cache"], x["v"])):
            if case["layout"] == "slots":
                cache[page, slot] = new[keep]
            else:
                cache[page, :, slot] = new[keep]
        return [q, x["k_cache"], x["v_cache"]]
    if kind == "attention":
        b, hq, d = x["q"].shape
        hk, lengths = case["kv_heads"], x["lengths"].long()
        pages = torch.clamp(x["pages"].long(), min=0)
        gathered = []
        for cache in (x["k_cache"], x["v_cache"]):
            t = cache[pages]                                                   # [sequence, page, ...]
            if case["layout"] == "heads":
                t = t.transpose(2, 3)
            gathered.append(t.reshape(b, -1, hk, d).permute(0, 2, 1, 3).float())   # [sequence, head, position, dim]
        k, v = gathered
        q = x["q"].float().reshape(b, hk, hq // hk, d)
        s = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
        there = torch.arange(s.shape[-1], device=s.device)[None, :] < lengths[:, None]
        s = torch.where(there[:, None, None, :], s, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(b, hq, d).to(dt)
    logits, target = x["logits"].float(), x["target"].long()
    counts = (target >= 0) & (target < case["vocab"])
    at = torch.where(counts, target, 0)[:, None]
    if kind == "logprob_grad":
        z = logits - x["lse"][:, None]
        p = torch.exp(z)
        dx = torch.where(p > 0, -p * (x["d_logprob"] * counts)[:, None] - p * (z + x["entropy"][:, None]) * x["d_entropy"][:, None], 0.0)
        dx.scatter_add_(1, at, (x["d_logprob"] * counts)[:, None])
        return dx.to(dt)
    m = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - m)
    total = e.sum(-1, keepdim=True)
    lse = (m + torch.log(total))[:, 0]
    entropy = lse - (torch.where(e > 0, e * logits, 0.0) / total).sum(-1)
    logprob = torch.where(counts, logits.gather(1, at)[:, 0] - lse, 0.0)
    if not case["top"]:
        return [logprob, lse, entropy]
    # unique keys: the value's order, then the lower index first
    bits = (logits + 0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7fffffff) - 1, bits) * 2 ** 32 + (2 ** 31 - 1 - torch.arange(case["vocab"], device=bits.device))
    ids = 2 ** 31 - 1 - (torch.topk(keys, case["top"], dim=-1).values & 0xffffffff)
    return [logprob, lse, entropy, logits.gather(1, ids) - lse[:, None], ids.int()]


def run(state):
    if not own:
        return _plain(state["case"], state["inputs"])
    args = state["args"]
    if state["case"]["kind"] == "append":
        out = state["thunk"](*args, donated=[False] * 8 + [True] * 2)
        args[8:] = out[1:]                        # the caches live on in the results
    else:
        out = state["thunk"](*args)
    return [_view(o) for o in out] if isinstance(out, tuple) else _view(out)


# ----------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------
def work(case):
    kind, e = case["kind"], _SIZE[case["dt"]]
    if kind == "embedding":
        n = float(case["tokens"]) * case["width"]
        return {"bytes": e * (_distinct(case) * float(case["width"]) + n) + 4.0 * case["tokens"], "flops": n}
    if kind == "embed_grad":
        n = float(case["tokens"]) * case["width"]
        return {"bytes": e * n + _SIZE[case["out"]] * float(case["rows"]) * case["width"] + 4.0 * case["tokens"], "flops": 2.0 * n}
    if kind == "append":
        t, d = float(case["tokens"]), case["head_dim"]
        turned = t * (case["q_heads"] + case["kv_heads"]) * case["rotary"]
        return {"bytes": 2 * e * t * d * (case["q_heads"] + 2 * case["kv_heads"]) + 4.0 * t * (case["rotary"] + 3), "flops": 3.0 * turned}
    if kind == "attention":
        n, b, d = float(sum(_lengths(case))), case["sequences"], case["head_dim"]
        return {"bytes": 2 * e * n * case["kv_heads"] * d + 2.0 * e * b * case["q_heads"] * d + 4.0 * (n / case["page"] + b),
                "flops": 4.0 * n * case["q_heads"] * d}
    n = float(case["tokens"]) * case["vocab"]
    if kind == "logprobs":
        return {"bytes": e * n + case["tokens"] * (16.0 + 8.0 * case["top"]), "flops": 5.0 * n}
    return {"bytes": 2 * e * n + 20.0 * case["tokens"], "flops": 6.0 * n}


# ----------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "embedding":
        table = torch.cat([x["table"].double() * case["scale"], torch.zeros((1, case["width"]), device="cuda", dtype=torch.float64)])
        return table[torch.where(x["ids"] < 0, case["rows"], x["ids"].long())]
    if kind == "embed_grad":
        out = torch.zeros((case["rows"] + 1, case["width"]), device="cuda", dtype=torch.float64)
        out.index_put_((torch.where(x["ids"] < 0, case["rows"], x["ids"].long()),), x["dy"].double(), accumulate=True)
        return out[:-1] * case["scale"]
    if kind == "append":
        position, half = x["position"].long(), case["rotary"] // 2
        there = position >= 0
        turn = torch.complex(x["cos"].double(), x["sin"].double())[position.clamp(min=0)][:, None, :]   # rotation = product with a unit number
        q, k = x["q"].double(), x["k"].double()
        for t in (q, k):
            if case["rotation"] == "halves":
                z = torch.complex(t[..., :half], t[..., half:2 * half]) * turn
                t[..., :half], t[..., half:2 * half] = z.real, z.imag
            else:
                z = torch.complex(t[..., 0:2 * half:2], t[..., 1:2 * half:2]) * turn
                t[..., 0:2 * half:2], t[..., 1:2 * half:2] = z.real, z.imag
        q[~there] = 0.0
        caches = [x["k_cache"].double(), x["v_cache"].double()]
        pages = x["pages"][x["sequence"].long()[there], position[there] // case["page"]].long()
        slots = position[there] % case["page"]
        for cache, new in zip(caches, (k, x["v"].double())):
            rows = cache if case["layout"] == "slots" else cache.permute(0, 2, 1, 3)
            rows.index_put_((pages, slots), new[there])
        return [q] + caches
    if kind == "attention":
        hk, g, d = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
        out = torch.zeros(x["q"].shape, device="cuda", dtype=torch.float64)
        for b, n in enumerate(x["lengths"].tolist()):
            pages = x["pages"][b, :-(-n // case["page"])].long()
            for h in range(hk if n else 0):
                k, v = ((c[pages, :, h] if case["layout"] == "slots" else c[pages, h]).reshape(-1, d)[:n].double() for c in (x["k_cache"], x["v_cache"]))
                w = torch.softmax(k @ x["q"][b, h * g:(h + 1) * g].double().t() / math.sqrt(d), 0)
                out[b, h * g:(h + 1) * g] = w.t() @ v
        return out
    n, v = case["tokens"], case["vocab"]
    parts = []
    for lo in range(0, n, 1024):
        logits, target = x["logits"][lo:lo + 1024].double(), x["target"][lo:lo + 1024].long()
        counts = target >= 0
        hot = torch.zeros_like(logits)
        hot[counts.nonzero()[:, 0], target[counts]] = 1.0
        if kind == "logprob_grad":
            z = logits - x["lse"][lo:lo + 1024, None].double()
            p = torch.exp(z)
            g, h = x["d_logprob"][lo:lo + 1024, None].double(), x["d_entropy"][lo:lo + 1024, None].double()
            parts.append(g * (hot - p * counts[:, None]) - h * torch.where(p > 0, p * (z + x["entropy"][lo:lo + 1024, None].double()), 0.0))
            continue
        lp = torch.log_softmax(logits, -1)
        res = [torch.where(hot > 0, lp, 0.0).sum(-1), torch.logsumexp(logits, -1), -torch.where(lp > -math.inf, torch.exp(lp) * lp, 0.0).sum(-1)]
        if case["top"]:
            values, ids, left = [], [], logits.clone()
            for _ in range(case["top"]):
                best = left.amax(-1, keepdim=True)
                first = torch.where(left == best, torch.arange(v, device="cuda"), v).amin(-1, keepdim=True)
                values.append(lp.gather(1, first))
                ids.append(first)
                left.scatter_(1, first, -math.inf)
            res += [torch.cat(values, 1), torch.cat(ids, 1).int()]
        parts.append(res)
    return torch.cat(parts) if kind == "logprob_grad" else [torch.cat(p) for p in zip(*parts)]
