"""Operators of a served language model, as they are measured.

Around its matrix products and its attention, one step of a model served with
8-bit activations, an 8-bit paged cache and drafted tokens runs

  rms_norm_e4m3   RMS norm of a residual stream, with the residual's addition,
                  into E4M3 codes and their scales (the operand of an 8-bit
                  product);
  cache_write     the new tokens' keys and values quantised into a paged cache;
  cache_read      sequences of that cache read back into dense rows;
  verify_draft    the drafted tokens accepted or rejected against the target's
                  probabilities, and one more token drawn.

`run` computes them in plain torch, or (with `own` true) with the calls of
libm3cuda.so's binding.  Codes are returned as float8_e4m3fn tensors beside
their scales.
"""

import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST = 448.0          # the largest E4M3 value
TINY = 2.0 ** -126       # the smallest scale: its reciprocal is finite
EPSILON = 1e-6


# ------------------------------------------------------------------- cases

def _norm(name, rows, width, group, dtype, residual):
    return dict(name=name, op="norm", rows=rows, width=width, group=group, dtype=dtype, residual=residual)


def _cache(name, op, sequences, tokens, context, page, heads, dim, dtype, strided=False):
    return dict(name=name, op=op, sequences=sequences, tokens=tokens, context=context, page=page, heads=heads,
                dim=dim, dtype=dtype, strided=strided)


def _verify(name, batch, drafts, vocabulary, dtype, draft, ragged):
    return dict(name=name, op="verify", batch=batch, drafts=drafts, vocabulary=vocabulary, dtype=dtype, draft=draft,
                ragged=ragged)


def listed():
    return [
        # one decoded token of one sequence: launch latency
        _norm("norm_one_token", 1, 2048, 2048, "bf16", True),
        # a chunk of a prompt, scales per 128 channels (block-scaled products)
        _norm("norm_chunk_groups", 1000, 5120, 128, "f16", False),
        # an odd width in full precision: no vector fits its rows
        _norm("norm_odd_width", 333, 2051, 2051, "f32", True),
        # a whole batch of prompts, the residual stream carried on
        _norm("norm_prefill", 16384, 4096, 4096, "bf16", True),
        # one new token for each of 32 sequences
        _cache("write_decode", "write", 32, 32, 1000, 16, 8, 128, "bf16"),
        # chunks of ragged length out of a fused projection's columns, odd heads and pages
        _cache("write_ragged", "write", 7, 3001, 500, 48, 5, 80, "f16", True),
        # a long prompt
        _cache("write_prompt", "write", 1, 16384, 0, 64, 8, 128, "bf16"),
        # a short sequence in full precision
        _cache("read_short", "read", 1, 500, 0, 16, 4, 64, "f32"),
        # the prefixes of 32 long sequences
        _cache("read_prefixes", "read", 32, 262144, 0, 64, 8, 128, "bf16"),
        # one sequence, four drafted tokens
        _verify("verify_one", 1, 4, 32000, "f32", True, False),
        # drafts without probabilities (looked up, not drawn), ragged, odd vocabulary
        _verify("verify_lookup_ragged", 24, 7, 50257, "bf16", False, True),
        # a large batch over a large vocabulary
        _verify("verify_batch", 128, 8, 131072, "f32", True, False),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "write", "read", "verify"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "norm":
        width = _log(rng, 64, 8192)
        if rng.random() < 0.7:
            width = max(64, width // 64 * 64)
        rows = _log(rng, 1, max(1, 16384 * 4096 * 2 // (width * SIZE[dtype])))
        groups = [width] + [g for g in (32, 64, 128) if width % g == 0]
        return dict(op=op, rows=min(rows, 32768), width=width, group=rng.choice(groups), dtype=dtype,
                    residual=rng.random() < 0.5)
    if op == "verify":
        drafts = rng.randint(1, 16)
        vocabulary = _log(rng, 1000, 131072)
        if rng.random() < 0.6:
            vocabulary = max(1000, vocabulary // 64 * 64)
        batch = _log(rng, 1, max(1, min(256, 128 * 8 * 131072 // (drafts * vocabulary))))
        return dict(op=op, batch=batch, drafts=drafts, vocabulary=vocabulary, dtype=dtype,
                    draft=rng.random() < 0.7, ragged=rng.random() < 0.5)
    heads, dim = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 80, 96, 128, 192, 256])
    most = (16384 if op == "write" else 262144) * 8 * 128 * 2 // (heads * dim * SIZE[dtype])
    tokens = _log(rng, 1, min(most, 65536))
    return dict(op=op, sequences=min(tokens, _log(rng, 1, 64)), tokens=tokens,
                context=rng.choice([0, rng.randint(1, 2000)]) if op == "write" else 0,
                page=rng.choice([1, 16, 24, 48, 64, 100, 256]), heads=heads, dim=dim, dtype=dtype,
                strided=op == "write" and rng.random() < 0.5)


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], SIZE[case["dtype"]]
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + 4 * n // case["group"] +
                case["width"] * size, "flops": 8 * n}
    if case["op"] == "verify":
        row = case["vocabulary"] * SIZE[case["dtype"]]
        return {"bytes": case["batch"] * (row * (2 if case["draft"] else 1) + case["drafts"] * 20 + 8),
                "flops": 3 * case["batch"] * case["vocabulary"]}
    vectors = 2 * case["tokens"] * case["heads"]
    return {"bytes": vectors * (case["dim"] * (SIZE[case["dtype"]] + 1) + 4) + 4 * case["tokens"] // case["page"],
            "flops": 3 * vectors * case["dim"]}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _norm_inputs(case, seed):
    """A residual stream: unit normals with a few channels far larger than the rest."""
    g, rows, width, t = _generator(seed), case["rows"], case["width"], DTYPES[case["dtype"]]
    channels = torch.where(torch.rand(width, generator=g, device="cuda") < 0.005, 20.0, 1.0)
    s = {"x": (_normal(g, rows, width) * channels).to(t), "w": (1 + 0.05 * _normal(g, width)).to(t)}
    if case["residual"]:
        s["r"] = (0.5 * _normal(g, rows, width)).to(t)
    return s


def _quantised(v):
    """E4M3 codes of float32 vectors along the last axis, and their scales."""
    scale = (v.abs().amax(-1) / LARGEST).clamp_min(TINY)
    return (v / scale[..., None]).to(torch.float8_e4m3fn), scale


def _cache_inputs(case, seed):
    """A batch of sequences over randomly placed pages, the cache as earlier steps left it, and the new tokens."""
    g, r = _generator(seed), np.random.RandomState(seed % (1 << 32))
    sequences, tokens, page, heads, dim = (case[k] for k in ("sequences", "tokens", "page", "heads", "dim"))
    cuts = np.sort(r.choice(tokens - 1, sequences - 1, replace=False) + 1) if sequences > 1 else np.empty(0, np.int64)
    offsets = np.concatenate([[0], cuts, [tokens]]).astype(np.int32)
    lengths = np.diff(offsets)
    starts = r.randint(0, case["context"] + 1, sequences).astype(np.int32)
    need = -(-(starts + lengths) // page)
    pages = (sequences * case["context"] + tokens) // page + sequences + 3
    order = r.permutation(pages).astype(np.int32)
    table = np.full((sequences, int(need.max())), -1, np.int32)
    at = 0
    for q in range(sequences):
        table[q, :need[q]] = order[at:at + need[q]]
        at += need[q]
    s = {"pages": pages}
    for name, a in (("offsets", offsets), ("starts", starts), ("table", table)):
        s[name] = torch.from_numpy(a).cuda()
    for name in ("key", "value"):
        channels = torch.exp(0.5 * _normal(g, heads, dim))
        codes, scales = _quantised(_normal(g, pages, page, heads, dim) * channels)
        s[name + "_codes"], s[name + "_scales"] = codes, scales
    if case["op"] == "write":
        t = DTYPES[case["dtype"]]
        if case["strided"]:  # the columns of one fused projection: queries, keys, values
            fused = _normal(g, tokens, 4 * heads, dim).to(t)
            s["keys"], s["values"] = fused[:, 2 * heads:3 * heads], fused[:, 3 * heads:]
        else:
            s["keys"], s["values"] = _normal(g, tokens, heads, dim).to(t), _normal(g, tokens, heads, dim).to(t)
    return s


def _verify_inputs(case, seed):
    """A target's probabilities, a draft model's that are near them, tokens drawn from the draft's."""
    g, t = _generator(seed), DTYPES[case["dtype"]]
    batch, drafts, vocabulary = case["batch"], case["drafts"], case["vocabulary"]
    logits = 2.5 * _normal(g, batch, drafts + 1, vocabulary)
    target = torch.softmax(logits, -1).to(t)
    logits = logits[:, :drafts] + 0.6 * _normal(g, batch, drafts, vocabulary)
    s = {"target": target, "uniforms": torch.rand(batch, drafts + 1, generator=g, device="cuda")}
    if case["draft"]:
        s["draft"] = torch.softmax(logits, -1).to(t)
    noise = torch.rand(batch, drafts, vocabulary, generator=g, device="cuda").clamp_min_(1e-20)
    s["tokens"] = (logits - torch.log(-torch.log(noise))).argmax(-1).to(torch.int32)
    if case["ragged"]:
        s["lengths"] = torch.randint(0, drafts + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    return s


def _inputs(case, seed):
    return {"norm": _norm_inputs, "write": _cache_inputs, "read": _cache_inputs, "verify": _verify_inputs}[case["op"]](
        case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _own_prepare(s)
    return s


# ------------------------------------------------------------- plain forms

def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    out = {}
    if "r" in s:
        out["sum"] = (x + s["r"].float()).to(s["x"].dtype)
        x = out["sum"].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * s["w"].float()
    codes, out["scales"] = _quantised(y.view(case["rows"], -1, case["group"]))
    out["codes"] = codes.view(y.shape)
    return out


def _slots(s):
    """The cache slot of each packed row."""
    case = s["case"]
    t = torch.arange(case["tokens"], device="cuda", dtype=torch.int32)
    q = torch.searchsorted(s["offsets"][1:], t, right=True)
    position = s["starts"][q] + t - s["offsets"][q]
    return s["table"][q, position // case["page"]].long() * case["page"] + position % case["page"]


def _plain_write(s):
    case, slots = s["case"], _slots(s)
    for new, name in (("keys", "key"), ("values", "value")):
        codes, scales = _quantised(s[new].float())
        s[name + "_codes"].view(torch.uint8).view(-1, case["heads"], case["dim"])[slots] = codes.view(torch.uint8)
        s[name + "_scales"].view(-1, case["heads"])[slots] = scales
    return {k: s[k] for k in ("key_codes", "key_scales", "value_codes", "value_scales")}


def _plain_read(s):
    case, slots, out = s["case"], _slots(s), {}
    for name in ("key", "value"):
        codes = s[name + "_codes"].view(torch.uint8).view(-1, case["heads"], case["dim"])[slots]
        scales = s[name + "_scales"].view(-1, case["heads"])[slots]
        out[name + "s"] = (codes.view(torch.float8_e4m3fn).float() * scales[..., None]).to(DTYPES[case["dtype"]])
    return out


def _plain_verify(s):
    case, target, tokens = s["case"], s["target"], s["tokens"].long()
    batch, drafts, device = case["batch"], case["drafts"], target.device
    place, rows = torch.arange(drafts, device=device), torch.arange(batch, device=device)
    lengths = s["lengths"].long() if "lengths" in s else torch.full((batch,), drafts, device=device)
    p = target[:, :drafts].gather(-1, tokens[..., None])[..., 0].double()
    q = s["draft"].gather(-1, tokens[..., None])[..., 0].double() if "draft" in s else torch.ones_like(p)
    fine = (s["uniforms"][:, :drafts].double() * q < p) & (place < lengths[:, None])
    accepted = fine.long().cumprod(-1).sum(-1)
    # the weights of the token drawn after the accepted ones; 64 bits, since a
    # draw next to a border of the running sum must fall on the same side
    p = target[rows, accepted].double()
    last = accepted.clamp_max(drafts - 1)
    if "draft" in s:
        q = s["draft"][rows, last].double()
    else:
        q = torch.zeros_like(p).scatter_(-1, tokens[rows, last][:, None], math.inf)
    w = torch.where((accepted < lengths)[:, None], (p - q).clamp_min(0), p)
    w = torch.where((w.sum(-1) > 0)[:, None], w, p)
    sums = w.cumsum(-1)
    drawn = (sums <= s["uniforms"][:, drafts, None].double() * sums[:, -1:]).sum(-1)
    place = torch.arange(drafts + 1, device=device)
    padded = torch.nn.functional.pad(tokens, (0, 1))
    out = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], drawn[:, None], -1))
    return {"tokens": out.int(), "accepted": accepted.int()}


# ------------------------------------------------- the framework's operators

def _package():
    name = "m3cuda"
    if name not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location(name, os.path.join(root, "m3.c_b200", "m3cuda.py"))
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


class _Device:
    """Device memory at `pointer` as torch sees other libraries' arrays; its owner lives as long as a tensor over it."""

    def __init__(self, owner, pointer, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": tuple(shape), "typestr": kind,
                                         "version": 2}


def _own_prepare(s):
    """What a program keeps from step to step: output buffers, the cache, the argument blocks that name them."""
    m3, case = _package(), s["case"]
    m3.load()
    dtype = {"f32": m3.F32, "f16": m3.F16, "bf16": m3.BF16}[case["dtype"]]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["codes"] = torch.empty(rows, width, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty(rows, width // case["group"], device="cuda")
        s["out"] = {"codes": s["codes"], "scales": s["scales"]}
        if "r" in s:
            s["out"]["sum"] = torch.empty_like(s["x"])
        s["args"] = m3.RmsNormE4m3Args(
            input=s["x"].data_ptr(), residual=s["r"].data_ptr() if "r" in s else None,
            sum=s["out"]["sum"].data_ptr() if "r" in s else None, dtype=dtype, scale=s["w"].data_ptr(),
            scale_dtype=dtype, rows=rows, width=width, group=case["group"], epsilon=EPSILON,
            codes=s["codes"].data_ptr(), code_scales=s["scales"].data_ptr())
    elif case["op"] == "verify":
        batch, drafts = case["batch"], case["drafts"]
        s["out"] = {"tokens": torch.empty(batch, drafts + 1, dtype=torch.int32, device="cuda"),
                    "accepted": torch.empty(batch, dtype=torch.int32, device="cuda")}
        s["args"] = m3.VerifyDraftArgs(
            target=s["target"].data_ptr(), draft=s["draft"].data_ptr() if "draft" in s else None, dtype=dtype,
            draft_tokens=s["tokens"].data_ptr(), lengths=s["lengths"].data_ptr() if "lengths" in s else None,
            uniforms=s["uniforms"].data_ptr(), batch=batch, drafts=drafts, vocabulary=case["vocabulary"],
            tokens=s["out"]["tokens"].data_ptr(), accepted=s["out"]["accepted"].data_ptr())
    else:
        heads, dim = case["heads"], case["dim"]
        cache = m3.Cache(pages=s["pages"], page_tokens=case["page"], heads=heads, head_dim=dim)
        shape = (s["pages"], case["page"], heads)
        views = {}
        for name, pointers in zip(("key", "value"), (cache.pointers()[:2], cache.pointers()[2:])):
            codes = torch.as_tensor(_Device(cache, pointers[0], shape + (dim,), "|u1"), device="cuda")
            views[name + "_codes"] = codes.view(torch.float8_e4m3fn)
            views[name + "_scales"] = torch.as_tensor(_Device(cache, pointers[1], shape, "<f4"), device="cuda")
        for name, view in views.items():
            view.copy_(s.pop(name))
        s["cache"] = cache
        s["batch"] = m3.CacheBatch(page_table=s["table"].data_ptr(), page_table_stride=s["table"].shape[1],
                                   offsets=s["offsets"].data_ptr(), starts=s["starts"].data_ptr(),
                                   sequences=case["sequences"], rows=case["tokens"])
        if case["op"] == "write":
            s["out"] = views
            k, v = s["keys"], s["values"]
        else:
            k, v = (torch.empty(case["tokens"], heads, dim, dtype=DTYPES[case["dtype"]], device="cuda")
                    for _ in range(2))
            s["out"] = {"keys": k, "values": v}
        s["rows"] = [m3.CacheRows(data=x.data_ptr(), dtype=dtype, token_stride=x.stride(0), head_stride=x.stride(1))
                     for x in (k, v)]
        torch.cuda.synchronize()


def _own_run(s):
    m3, op = sys.modules["m3cuda"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        m3.rms_norm_e4m3(s["args"], device=0, stream=stream)
    elif op == "verify":
        m3.verify_draft(s["args"], device=0, stream=stream)
    elif op == "write":
        s["cache"].write(s["batch"], s["rows"][0], s["rows"][1], stream=stream)
    else:
        s["cache"].read(s["batch"], s["rows"][0], s["rows"][1], stream=stream)
    return s["out"]


def run(state):
    if own:
        return _own_run(state)
    return {"norm": _plain_norm, "write": _plain_write, "read": _plain_read, "verify": _plain_verify}[
        state["case"]["op"]](state)


# ----------------------------------------------- the definition, in 64 bits

def _nearest_e4m3(v):
    """The E4M3 value nearest to v (ties to the even significand), |v| <= 448."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_(-6, 8)
    exponent = torch.where(torch.ldexp(torch.ones_like(v), exponent + 1) <= v.abs(), exponent + 1, exponent)
    exponent = torch.where(torch.ldexp(torch.ones_like(v), exponent) > v.abs(), exponent - 1, exponent).clamp_(-6, 8)
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return (torch.round(v / step) * step).clamp_(-LARGEST, LARGEST)


def _exact_codes(v):
    scale = torch.clamp(torch.amax(torch.abs(v), dim=-1, keepdim=True) / LARGEST, min=TINY)
    return _nearest_e4m3(v / scale), scale.squeeze(-1)


def _exact_slots(s, case):
    offsets, starts, table = (s[k].cpu().numpy().astype(np.int64) for k in ("offsets", "starts", "table"))
    slots = np.empty(case["tokens"], np.int64)
    for q in range(case["sequences"]):
        position = starts[q] + np.arange(offsets[q + 1] - offsets[q])
        slots[offsets[q]:offsets[q + 1]] = table[q][position // case["page"]] * case["page"] + position % case["page"]
    return torch.from_numpy(slots).cuda()


def _exact_norm(s, case):
    out, x = {}, s["x"].double()
    if "r" in s:
        # the stored sum is a rounded value, and the norm's input
        out["sum"] = x + s["r"].double()
        x = out["sum"].to(s["x"].dtype).double()
    y = x * s["w"].double() / torch.sqrt((x * x).sum(-1, keepdim=True) / case["width"] + EPSILON)
    codes, out["scales"] = _exact_codes(y.reshape(case["rows"], case["width"] // case["group"], case["group"]))
    out["codes"] = codes.reshape(case["rows"], case["width"])
    return out


def _exact_verify(s, case):
    drafts, place = case["drafts"], np.full((case["batch"], case["drafts"] + 1), -1, np.int32)
    tokens, uniforms = s["tokens"].cpu().numpy(), s["uniforms"].cpu().numpy().astype(np.float64)
    count = np.zeros(case["batch"], np.int32)
    for b in range(case["batch"]):
        length = int(s["lengths"][b]) if "lengths" in s else drafts
        m = 0
        while m < length:
            d = tokens[b, m]
            q = float(s["draft"][b, m, d]) if "draft" in s else 1.0
            if not uniforms[b, m] * q < float(s["target"][b, m, d]):
                break
            place[b, m] = d
            m += 1
        p = s["target"][b, m].double().cpu().numpy()
        w = p
        if m < length:
            if "draft" in s:
                w = np.maximum(p - s["draft"][b, m].double().cpu().numpy(), 0)
            else:
                w = p.copy()
                w[tokens[b, m]] = 0
            w = w if w.any() else p
        sums = np.cumsum(w)
        place[b, m] = np.searchsorted(sums, uniforms[b, drafts] * sums[-1], side="right")
        count[b] = m
    return {"tokens": torch.from_numpy(place), "accepted": torch.from_numpy(count)}


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "norm":
        return _exact_norm(s, case)
    if op == "verify":
        return _exact_verify(s, case)
    slots, out = _exact_slots(s, case), {}
    for new, name in (("keys", "key"), ("values", "value")):
        codes, scales = s[name + "_codes"].double(), s[name + "_scales"].double()
        if op == "read":
            out[new] = codes.view(-1, case["heads"], case["dim"])[slots]
            out[new] *= scales.view(-1, case["heads"])[slots].unsqueeze(-1)
        else:
            c, a = _exact_codes(s[new].double())
            codes.view(-1, case["heads"], case["dim"])[slots] = c
            scales.view(-1, case["heads"])[slots] = a
            out[name + "_codes"], out[name + "_scales"] = codes, scales
    return out
