"""The serving operators around a paged key-value cache, as cases that can be timed and checked.

Three operators: the append of new keys and values to a paged cache with the position
rotation of q and k applied on the way, attention of one new token per sequence over that
cache, and attention over whole packed prompts.  Each has a plain form in elementary torch
operations in 32 bits (`own` false) and the library's call (`own` true), on the same state.
Head layouts are those of the library's model configurations: 32 query and 8 key-value
heads of 64 or 128, 64 and 8 of 128, and one eighth of the last (a tensor-parallel shard).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LAYOUTS = [(32, 8, 64), (32, 8, 128), (64, 8, 128), (8, 1, 128)]
ROPE_BASE = 500000.0


def listed():
    return [
        # a decode step of a 64-sequence batch: one new token each, latency counts
        {"name": "append_step_bf16", "op": "append", "heads": 32, "kv_heads": 8, "head_dim": 128, "batch": 64,
         "low": 1, "high": 1, "past": 3000, "page": 16, "kind": "bf16", "inputs": "bf16", "queries": "bf16",
         "style": "pairs", "mix": 1},
        # packed prompts from f32 projections, halves of a head rotated against each other
        {"name": "append_prompts_f16", "op": "append", "heads": 32, "kv_heads": 8, "head_dim": 128, "batch": 7,
         "low": 500, "high": 2000, "past": 0, "page": 64, "kind": "f16", "inputs": "f32", "queries": "f16",
         "style": "halves", "mix": 2},
        # ragged chunks into a Q8_0 cache
        {"name": "append_chunks_q8_0", "op": "append", "heads": 32, "kv_heads": 8, "head_dim": 64, "batch": 9,
         "low": 1, "high": 400, "past": 700, "page": 32, "kind": "q8_0", "inputs": "f16", "queries": "f16",
         "style": "pairs", "mix": 3},
        # one chat of some hundred tokens: the smallest call
        {"name": "decode_one_short_f16", "op": "decode", "heads": 32, "kv_heads": 8, "head_dim": 64, "batch": 1,
         "low": 777, "high": 777, "page": 16, "kind": "f16", "queries": "f16", "mix": 4},
        # one very long context: the work has to be split over its length
        {"name": "decode_one_long_bf16", "op": "decode", "heads": 64, "kv_heads": 8, "head_dim": 128, "batch": 1,
         "low": 131071, "high": 131071, "page": 64, "kind": "bf16", "queries": "bf16", "mix": 5},
        # a continuous batch with lengths from one token to eight thousand
        {"name": "decode_ragged_bf16", "op": "decode", "heads": 32, "kv_heads": 8, "head_dim": 128, "batch": 64,
         "low": 1, "high": 8192, "page": 16, "kind": "bf16", "queries": "bf16", "mix": 6},
        # the same kind of batch over a Q8_0 cache
        {"name": "decode_ragged_q8_0", "op": "decode", "heads": 32, "kv_heads": 8, "head_dim": 128, "batch": 48,
         "low": 300, "high": 6000, "page": 32, "kind": "q8_0", "queries": "f16", "mix": 7},
        # three short prompts: the smallest prompt call
        {"name": "prompt_short_bf16", "op": "prompt", "heads": 32, "kv_heads": 8, "head_dim": 64, "batch": 3,
         "low": 5, "high": 61, "past": 0, "kind": "bf16", "causal": True, "mix": 8},
        # many prompts of different lengths in one call
        {"name": "prompt_ragged_f16", "op": "prompt", "heads": 32, "kv_heads": 8, "head_dim": 64, "batch": 12,
         "low": 17, "high": 2048, "past": 0, "kind": "f16", "causal": True, "mix": 9},
        # chunks of prompts whose first part is already known: more keys than queries
        {"name": "prompt_chunks_bf16", "op": "prompt", "heads": 64, "kv_heads": 8, "head_dim": 128, "batch": 4,
         "low": 300, "high": 512, "past": 4000, "kind": "bf16", "causal": True, "mix": 10},
        # one long prompt: the largest call
        {"name": "prompt_long_bf16", "op": "prompt", "heads": 32, "kv_heads": 8, "head_dim": 128, "batch": 1,
         "low": 8192, "high": 8192, "past": 0, "kind": "bf16", "causal": True, "mix": 11},
    ]


def spread(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice(LAYOUTS)
    case = {"op": rng.choice(["append", "decode", "prompt"]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "mix": rng.randrange(1 << 20)}
    if case["op"] == "append":
        high = spread(rng, 1, 2000)
        case.update(batch=spread(rng, 1, max(1, 7000 // high)) if high > 1 else spread(rng, 1, 256), low=1, high=high,
                    past=rng.choice([0, spread(rng, 1, 4000)]), page=rng.choice([8, 16, 32, 64, 128]),
                    kind=rng.choice(["f16", "bf16", "q8_0"]), inputs=rng.choice(["f32", "f16", "bf16"]),
                    queries=rng.choice(["f16", "bf16"]), style=rng.choice(["pairs", "halves"]))
        if heads == 64:
            case["batch"] = max(1, case["batch"] // 2)
    elif case["op"] == "decode":
        kind = rng.choice(["f16", "bf16", "q8_0"])
        high = spread(rng, 1, 131072)
        case.update(batch=spread(rng, 1, max(1, min(256, 250000 // high))), low=rng.choice([1, high]), high=high,
                    page=rng.choice([8, 16, 32, 64, 128]), kind=kind,
                    queries=rng.choice(["f16", "bf16"]) if kind == "q8_0" else kind)
    else:
        high = spread(rng, 1, 4000)
        case.update(batch=spread(rng, 1, max(1, min(32, (3500 // high) ** 2))), low=rng.choice([1, high]), high=high,
                    past=rng.choice([0, 0, spread(rng, 1, 4000)]), kind=rng.choice(["f16", "bf16"]),
                    causal=rng.random() < 0.8)
    return case


def lengths_of(case):
    """New tokens (append, prompt) or cached tokens (decode) of each sequence, and the tokens before them."""
    rng = random.Random(case["mix"])
    lens = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    past = [rng.randint(case["past"] // 2, case["past"]) for _ in lens] if case.get("past") else [0 for _ in lens]
    return lens, past


def starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def cache(case, gen, pages):
    """A cache with earlier contents in every page: values, or int8 values and f16 scales of 32 each."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    if case["kind"] != "q8_0":
        return [normal(shape, gen, DTYPES[case["kind"]]) for _ in range(2)] + [None, None]
    values = [torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8) for _ in range(2)]
    shape = shape[:3] + (case["head_dim"] // 32,)
    return values + [(torch.rand(shape, generator=gen, device="cuda") * 0.01 + 0.01).half() for _ in range(2)]


def paging(case, gen, totals):
    """A page table over randomly placed pages, some pages left free."""
    width = max(1, max(-(-n // case["page"]) for n in totals))
    used = sum(-(-n // case["page"]) for n in totals)
    pages = used + used // 16 + 1
    order = torch.randperm(pages, generator=gen, device="cuda")[:used].to(torch.int32)
    counts = torch.tensor([-(-n // case["page"]) for n in totals], device="cuda")
    first = counts.cumsum(0) - counts
    column = torch.arange(width, device="cuda")
    inside = column < counts[:, None]
    table = torch.where(inside, order[(first[:, None] + column).clamp(max=used - 1)], 0).to(torch.int32).contiguous()
    return table, width, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, past = lengths_of(case)
    heads, kv_heads, head_dim = case["heads"], case["kv_heads"], case["head_dim"]
    state = {"case": case, "batch": case["batch"], "scale": head_dim ** -0.5}
    if case["op"] == "append":
        totals = [a + b for a, b in zip(lens, past)]
        tokens, kind = sum(lens), DTYPES[case["inputs"]]
        state["table"], state["width"], pages = paging(case, gen, totals)
        state["k"], state["v"], state["k_scales"], state["v_scales"] = cache(case, gen, pages)
        # q, k and v as one projection leaves them: side by side in a row of one token
        rows = normal((tokens, heads + 2 * kv_heads, head_dim), gen, kind)
        state["rows"], state["tokens"], state["pages"] = rows, tokens, pages
        state["cu"], state["lengths"] = ints(starts(lens)), ints(totals)
        state["rope_len"] = max(totals)
        angles = torch.arange(max(totals), device="cuda", dtype=torch.float64)[:, None] * ROPE_BASE ** (
            -torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float64) / head_dim)
        state["rope"] = torch.stack([angles.sin(), angles.cos()], -1).float()
        state["out"] = torch.zeros((tokens, heads, head_dim), dtype=DTYPES[case["queries"]], device="cuda")
    elif case["op"] == "decode":
        state["table"], state["width"], pages = paging(case, gen, lens)
        state["k"], state["v"], state["k_scales"], state["v_scales"] = cache(case, gen, pages)
        state["pages"], state["lengths"] = pages, ints(lens)
        state["q"] = normal((case["batch"], heads, head_dim), gen, DTYPES[case["queries"]], 1.5)
        state["out"] = torch.zeros_like(state["q"])
    else:
        totals, kind = [a + b for a, b in zip(lens, past)], DTYPES[case["kind"]]
        state["tokens"], state["keys"] = sum(lens), sum(totals)
        state["max_q"], state["max_k"] = max(lens), max(totals)
        state["cu_q"], state["cu_k"] = ints(starts(lens)), ints(starts(totals))
        state["q"] = normal((sum(lens), heads, head_dim), gen, kind, 1.5)
        state["k"] = normal((sum(totals), kv_heads, head_dim), gen, kind)
        state["v"] = normal((sum(totals), kv_heads, head_dim), gen, kind)
        state["out"] = torch.zeros_like(state["q"])
    if own:
        import nanocamelid_b200 as ncm
        types = {"f32": ncm.F32, "f16": ncm.F16, "bf16": ncm.BF16, "q8_0": ncm.Q8_0}
        state["ncm"] = ncm
        state["types"] = {k: types[case[k]] for k in ("kind", "inputs", "queries") if k in case}
        if case["op"] != "prompt":
            state["kv"] = ncm.PagedKV(types[case["kind"]], state["k"].data_ptr(), state["v"].data_ptr(), pages,
                                      case["page"], kv_heads, head_dim,
                                      state["k_scales"].data_ptr() if case["kind"] == "q8_0" else 0,
                                      state["v_scales"].data_ptr() if case["kind"] == "q8_0" else 0)
        if case["op"] == "decode":
            size = ncm.paged_attention_workspace(heads, kv_heads, head_dim)
            state["space"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------- the plain forms
def rotate(x, s, c, style):
    """x [tokens, heads, dim] turned by the angles whose sines and cosines are s and c [tokens, 1, dim / 2]."""
    if style == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def toward_zero_f16(x):
    """f32 values that are not negative, as f16 rounded toward zero."""
    h = x.half()
    return torch.where(h.float() > x, (h.view(torch.int16) - 1).view(torch.float16), h)


def quantised(x):
    """Q8_0 of blocks of 32 along the last axis: the largest magnitude / 127 is the scale (kept as f16, rounded toward
    zero), a value is x times the scale's reciprocal rounded to the nearest whole number, halves away from zero."""
    blocks = x.unflatten(-1, (-1, 32))
    scale = blocks.abs().amax(-1) / 127.0
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    y = (blocks * inverse[..., None]).double()   # the half that is added below would be rounded in 32 bits
    whole = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127)
    return whole.to(torch.int8).flatten(-2), toward_zero_f16(scale)


def values_of(ints8, scales):
    """The values that a Q8_0 cache holds, in f32."""
    return (ints8.unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def append_outputs(state):
    if state["case"]["kind"] == "q8_0":
        return {"q": state["out"], "k": values_of(state["k"], state["k_scales"]),
                "v": values_of(state["v"], state["v_scales"])}
    return {"q": state["out"], "k": state["k"], "v": state["v"]}


def plain_append(state):
    case, cu = state["case"], state["cu"].long()
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    token = torch.arange(state["tokens"], device="cuda")
    seq = torch.bucketize(token, cu[1:], right=True)
    pos = state["lengths"].long()[seq] - cu[seq + 1] + token
    where, off = state["table"].long()[seq, pos // page], pos % page
    q, k, v = state["rows"].float().split([heads, kv_heads, kv_heads], 1)
    s, c = state["rope"][pos].unbind(-1)
    s, c = s[:, None], c[:, None]
    state["out"].copy_(rotate(q, s, c, case["style"]))
    for x, name in ((rotate(k, s, c, case["style"]), "k"), (v, "v")):
        if case["kind"] == "q8_0":
            x, scales = quantised(x)
            state[name + "_scales"][where, :, off] = scales
        state[name][where, :, off] = x.to(state[name].dtype)
    return append_outputs(state)


def gathered(state, name):
    """A cache's rows in their sequences' order, [batch, kv_heads, width * page, dim], in f32."""
    x = state[name][state["table"].long()]
    if state["case"]["kind"] == "q8_0":
        x = values_of(x, state[name + "_scales"][state["table"].long()])
    return x.float().transpose(1, 2).flatten(2, 3)


def weighted(scores, mask, values):
    """Softmax of the scores where the mask is true (all zeros where it leaves nothing), times the values."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    return (weights @ values) / total.where(total > 0, 1.0)


def plain_decode(state):
    case = state["case"]
    k, v = gathered(state, "k"), gathered(state, "v")
    q = state["q"].float().unflatten(1, (case["kv_heads"], -1))
    mask = torch.arange(k.shape[2], device="cuda") < state["lengths"][:, None]
    out = weighted((q @ k.transpose(2, 3)) * state["scale"], mask[:, None, None], v)
    return state["out"].copy_(out.flatten(1, 2))


def plain_prompt(state):
    case = state["case"]
    cu_q, cu_k = state["cu_q"].long(), state["cu_k"].long()
    n_q, n_k = cu_q.diff(), cu_k.diff()
    at_q, at_k = torch.arange(state["max_q"], device="cuda"), torch.arange(state["max_k"], device="cuda")
    has_q, has_k = at_q < n_q[:, None], at_k < n_k[:, None]
    rows_q = (cu_q[:-1, None] + at_q).where(has_q, 0)
    rows_k = (cu_k[:-1, None] + at_k).where(has_k, 0)
    q = state["q"][rows_q].float().unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (state[x][rows_k].float().transpose(1, 2) for x in ("k", "v"))
    scores = ((q @ k.transpose(2, 3)) * state["scale"]).unflatten(2, (-1, state["max_q"]))
    mask = has_k[:, None, :]
    if case["causal"]:   # the last query sees the last key
        mask = mask & (at_k <= (at_q + (n_k - n_q)[:, None])[:, :, None])
    out = weighted(scores, mask[:, None, None], v[:, :, None]).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return state["out"].copy_(out[has_q])


# ---------------------------------------------------------------- the library's calls
def own_append(state):
    case, rows, types = state["case"], state["rows"], state["types"]
    heads, kv_heads, head_dim = case["heads"], case["kv_heads"], case["head_dim"]
    ncm, at, wide = state["ncm"], rows.data_ptr(), rows.element_size() * head_dim
    stride = (heads + 2 * kv_heads) * head_dim
    ncm.paged_append(state["kv"], types["inputs"], at, at + wide * heads, at + wide * (heads + kv_heads),
                     state["out"].data_ptr(), types["queries"], state["tokens"], heads, state["batch"],
                     state["cu"].data_ptr(), state["lengths"].data_ptr(), state["table"].data_ptr(), state["width"],
                     rope_ptr=state["rope"].data_ptr(), rope_len=state["rope_len"], rope_half=head_dim // 2,
                     rope_style=ncm.ROPE_PAIRS if case["style"] == "pairs" else ncm.ROPE_HALVES, q_stride=stride,
                     k_stride=stride, v_stride=stride, stream=torch.cuda.current_stream().cuda_stream)
    return append_outputs(state)


def own_decode(state):
    case, out, space = state["case"], state["out"], state["space"]
    state["ncm"].paged_attention(out.data_ptr(), state["q"].data_ptr(), state["kv"], state["types"]["queries"],
                                 state["batch"], case["heads"], state["lengths"].data_ptr(), state["table"].data_ptr(),
                                 state["width"], space.data_ptr(), space.numel(), scale=state["scale"],
                                 stream=torch.cuda.current_stream().cuda_stream)
    return out


def own_prompt(state):
    case, out = state["case"], state["out"]
    state["ncm"].prompt_attention(out.data_ptr(), state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(),
                                  state["types"]["kind"], state["tokens"], state["keys"], state["batch"],
                                  case["heads"], case["kv_heads"], case["head_dim"], state["cu_q"].data_ptr(),
                                  state["cu_k"].data_ptr(), causal=case["causal"], scale=state["scale"],
                                  stream=torch.cuda.current_stream().cuda_stream)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return own_append(state) if op == "append" else own_decode(state) if op == "decode" else own_prompt(state)
    return plain_append(state) if op == "append" else plain_decode(state) if op == "decode" else plain_prompt(state)


# ---------------------------------------------------------------- the work, and the values in 64 bits
def work(case):
    lens, past = lengths_of(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "q8_0": 34 / 32}
    if case["op"] == "append":
        tokens = sum(lens)
        places = max(a + b for a, b in zip(lens, past)) if not any(past) else tokens   # rows of the rotation table
        moved = tokens * dim * ((heads + 2 * kv_heads) * size[case["inputs"]] + heads * size[case["queries"]]
                                + 2 * kv_heads * size[case["kind"]]) + min(places, tokens) * dim * 4
        return {"bytes": int(moved), "flops": 3 * tokens * dim * (heads + kv_heads)}
    if case["op"] == "decode":
        keys = sum(lens)
        moved = 2 * keys * kv_heads * dim * size[case["kind"]] + 2 * case["batch"] * heads * dim * 2
        return {"bytes": int(moved), "flops": 4 * keys * heads * dim}
    pairs = sum(n * (n + 1) // 2 + n * p if case["causal"] else n * (n + p) for n, p in zip(lens, past))
    totals = sum(lens) + sum(past)
    return {"bytes": 2 * dim * (2 * sum(lens) * heads + 2 * totals * kv_heads), "flops": 4 * pairs * heads * dim}


def attention64(q, k, v, scale, offset):
    """One sequence in 64 bits: q [n, heads, dim], k and v [m, kv_heads, dim]; query i sees keys up to i + offset
    (all of them where offset is None)."""
    n, heads, dim = q.shape
    out = torch.zeros((n, heads, dim), dtype=torch.float64, device=q.device)
    group = heads // k.shape[1]
    for h in range(heads):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        for i in range(0, n, 4096):
            s = torch.einsum("id,jd->ij", q[i:i + 4096, h].double(), kh) * scale
            if offset is not None:
                last = torch.arange(i, i + s.shape[0], device=q.device) + offset
                s[torch.arange(s.shape[1], device=q.device)[None] > last[:, None]] = -math.inf
            out[i:i + 4096, h] = torch.softmax(s, -1).nan_to_num(0.0) @ vh if s.shape[1] else 0.0
    return out


def exact(case, seed):
    state = prepare(case, seed)
    lens, past = lengths_of(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prompt":
        at, ak = starts(lens), starts([a + b for a, b in zip(lens, past)])
        return torch.cat([attention64(state["q"][at[i]:at[i + 1]], state["k"][ak[i]:ak[i + 1]],
                                      state["v"][ak[i]:ak[i + 1]], state["scale"], past[i] if case["causal"] else None)
                          for i in range(len(lens))])
    table = state["table"].cpu()
    if case["op"] == "decode":
        rows = []
        for i, n in enumerate(lens):
            pages = table[i, :-(-n // case["page"])].long().cuda()
            kv = []
            for name in ("k", "v"):
                x = state[name][pages].double()
                if case["kind"] == "q8_0":
                    x = x * state[name + "_scales"][pages].double().repeat_interleave(32, -1)
                kv.append(x.permute(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:n])
            rows.append(attention64(state["q"][i:i + 1], kv[0], kv[1], state["scale"], None))
        return torch.cat(rows)
    positions = torch.cat([torch.arange(p, p + n) for n, p in zip(lens, past)]).cuda()
    x = state["rows"].double()
    turn = torch.complex(state["rope"][positions, :, 1].double(), state["rope"][positions, :, 0].double())[:, None]
    turned = x[:, :heads + kv_heads]
    if case["style"] == "pairs":
        y = torch.view_as_real(torch.view_as_complex(turned.reshape(*turned.shape[:2], -1, 2).contiguous()) * turn)
        y = y.reshape(turned.shape)
    else:
        z = torch.complex(turned[..., :dim // 2].contiguous(), turned[..., dim // 2:].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    if case["kind"] == "q8_0":   # what is held in 8 bits has no value of its own in 64
        return {"q": y[:, :heads], "k": None, "v": None}
    k, v = state["k"].double(), state["v"].double()
    at = starts(lens)
    for i, n in enumerate(lens):
        place = torch.arange(past[i], past[i] + n)
        pages, off = table[i].long()[place // case["page"]].cuda(), (place % case["page"]).cuda()
        k[pages, :, off] = y[at[i]:at[i + 1], heads:]
        v[pages, :, off] = x[at[i]:at[i + 1], heads + kv_heads:]
    return {"q": y[:, :heads], "k": k, "v": v}
