"""The text-conditioning operators of fp8_b200, as work to be timed and compared.

Three operators carry a prompt into the UNet: the token embedding with its
gradient by sorted tokens, dropout whose mask comes from a counter and is never
stored, and the attention of the image's queries over the encoder's states.
Each case is one pass of one of them, in its plain form (elementary torch
operations in 32 bits) or through the framework's entry points (``own``).
"""

from __future__ import annotations

import math
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------ cases
def _attend(name, b, lq, lk, heads, kv_heads, dim, dtype, mask, packed, train):
    return {"name": name, "op": "attend", "b": b, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "mask": mask, "packed": packed, "train": train}


def _embed(name, tokens, vocab, width, wdtype, dtype, ids, padding, train):
    return {"name": name, "op": "embed", "tokens": tokens, "vocab": vocab, "width": width, "wdtype": wdtype,
            "dtype": dtype, "ids": ids, "padding": padding, "train": train}


def _dropout(name, rows, width, dtype, p, residual, train):
    return {"name": name, "op": "dropout", "rows": rows, "width": width, "dtype": dtype, "p": p,
            "residual": residual, "train": train}


def listed():
    return [
        # one new token against one sequence's encoder states: the smallest call of a server
        _attend("attend_one_token", 1, 1, 1024, 4, 4, 64, "bf16", "none", False, False),
        # a batch of single tokens with grouped heads over long states of many lengths
        _attend("attend_token_batch", 32, 1, 8192, 16, 4, 128, "bf16", "lengths", False, False),
        # the UNet's 16x16 attention resolution (256 queries, 4 heads of 64, batch 128) over prompts of up to
        # 77 tokens, in training
        _attend("attend_prompt_train", 128, 256, 77, 4, 4, 64, "bf16", "lengths", True, True),
        # sampling at 32x32 pixels (1024 queries) over contexts of up to 256 tokens
        _attend("attend_prompt_sample", 64, 1024, 256, 4, 4, 64, "bf16", "lengths", True, False),
        # long queries over long states, heads of 128, in training: the largest
        _attend("attend_long_train", 2, 4096, 4096, 8, 8, 128, "bf16", "none", False, True),
        # odd sizes, grouped heads of 80, a key mask with holes that leaves one sequence nothing
        _attend("attend_ragged_train", 5, 333, 1021, 8, 2, 80, "fp16", "mask", False, True),
        # one prompt's tokens for sampling
        _embed("embed_prompt", 77, 32768, 512, "fp32", "bf16", "frequent", False, False),
        # a training batch of 128 prompts of 77 tokens, most of them frequent words or padding
        _embed("embed_prompt_train", 128 * 77, 32768, 512, "fp32", "bf16", "frequent", True, True),
        # a long-text batch over a large vocabulary of bf16 weights
        _embed("embed_long_train", 262147, 131072, 1024, "bf16", "bf16", "frequent", False, True),
        # dropout of one prompt's embedding
        _dropout("dropout_prompt", 77, 512, "bf16", 0.1, False, False),
        # dropout of a block's output onto its residual: 128 images of 32x32 pixels of 128 channels
        _dropout("dropout_join_train", 128 * 1024, 128, "bf16", 0.1, True, True),
        # a long batch in 32 bits, an odd number of elements
        _dropout("dropout_long_train", 16385, 4093, "fp32", 0.25, False, True),
    ]


MOST = {"attend": (14 * 2 * 8 * 4096 * 4096 * 128, 2 * 32 * 8192 * 4 * 128 * 2, 2 * 8 * 4096 * 4096),
        "embed": (0, 262147 * 1024 * 8 + 131072 * 1024 * 4, 262147 * 1024),
        "dropout": (0, 16385 * 4093 * 16, 16385 * 4093)}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw(rng):
    op = rng.choice(["attend", "attend", "embed", "dropout"])
    if op == "attend":
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        group = rng.choice([1, 1, 2, 3, 4])
        train = rng.random() < 0.5
        lq = 1 if not train and rng.random() < 0.4 else _log(rng, 2, 4096)
        return _attend("", _log(rng, 1, 128), lq, _log(rng, 1, 8192), kv_heads * group, kv_heads,
                       rng.choice([32, 40, 64, 64, 80, 96, 128]), rng.choice(["bf16", "bf16", "fp16"]),
                       rng.choice(["none", "lengths", "mask"]), rng.random() < 0.5, train)
    if op == "embed":
        return _embed("", _log(rng, 1, 262147), _log(rng, 100, 131072), rng.choice([64, 250, 256, 512, 777, 1024]),
                      rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["fp32", "bf16", "fp16"]),
                      rng.choice(["frequent", "uniform"]), rng.random() < 0.5, rng.random() < 0.7)
    return _dropout("", _log(rng, 1, 131072), rng.choice([63, 128, 256, 512, 777, 1024, 4093]),
                    rng.choice(["fp32", "bf16", "fp16"]), rng.choice([0.05, 0.1, 0.25, 0.5]), rng.random() < 0.5,
                    rng.random() < 0.6)


def draw(rng):
    while True:
        case = _draw(rng)
        flops, size, cells = MOST[case["op"]]
        need = work(case)
        here = {"attend": lambda c: c["b"] * c["heads"] * c["lq"] * c["lk"],
                "embed": lambda c: c["tokens"] * c["width"],
                "dropout": lambda c: c["rows"] * c["width"]}[case["op"]](case)
        if need["bytes"] <= size and (not flops or need["flops"] <= flops) and here <= cells:
            del case["name"]
            return case


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Key counts from a quarter of the states to all of them, evenly spread over the batch."""
    b, lk = case["b"], case["lk"]
    return [max(1, lk - (3 * lk * i) // (4 * b)) for i in range(b)]


def _kept(case):
    """Keys each sequence keeps under the key mask: four of five; the first sequence of several keeps none."""
    b, lk = case["b"], case["lk"]
    return [0 if b > 1 and i == 0 else max(1, (4 * lk) // 5) for i in range(b)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape, dtype: torch.randn(*shape, generator=g, device=dev).to(dtype)  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    st = dict(case)
    if case["op"] == "attend":
        b, lq, lk, h, hkv, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
        # layer-normed activations through a projection: about unit variance
        st["q"] = randn(b, lq, h, d, dtype=dtype).requires_grad_(case["train"])
        if case["packed"]:  # one projection of the encoder's states gives keys and values side by side
            st["kv"] = randn(b, lk, 2, hkv, d, dtype=dtype).requires_grad_(case["train"])
        else:
            st["k"] = randn(b, lk, hkv, d, dtype=dtype).requires_grad_(case["train"])
            st["v"] = randn(b, lk, hkv, d, dtype=dtype).requires_grad_(case["train"])
        st["key_lengths"] = st["key_mask"] = None
        if case["mask"] == "lengths":
            order = torch.randperm(b, generator=g, device=dev)
            st["key_lengths"] = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)[order]
        elif case["mask"] == "mask":
            rank = torch.rand(b, lk, generator=g, device=dev).argsort(dim=1).argsort(dim=1)
            st["key_mask"] = rank < torch.tensor(_kept(case), device=dev)[:, None]
        if case["train"]:
            st["dout"] = randn(b, lq, h, d, dtype=dtype)
    elif case["op"] == "embed":
        n, vocab, width = case["tokens"], case["vocab"], case["width"]
        u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
        if case["ids"] == "frequent":  # a few tokens are very frequent, most are rare
            ids = (float(vocab) ** u).long() - 1
        else:
            ids = (u * vocab).long()
        if case["padding"]:  # the ends of the prompts are the padding token
            ids[torch.rand(n, generator=g, device=dev) < 0.3] = 0
        st["token_ids"] = ids.clamp_(0, vocab - 1)
        st["padding_idx"] = 0 if case["padding"] else None
        st["scale"] = math.sqrt(width)
        st["weight"] = (randn(vocab, width, dtype=torch.float32) / math.sqrt(width)).to(DTYPES[case["wdtype"]])
        st["weight"].requires_grad_(case["train"])
        if case["train"]:
            st["dout"] = randn(n, width, dtype=dtype)
    else:
        rows, width = case["rows"], case["width"]
        st["x"] = randn(rows, width, dtype=dtype).requires_grad_(case["train"])
        st["seed"] = torch.randint(-2**62, 2**62, (), generator=g, device=dev, dtype=torch.int64)
        st["add"] = randn(rows, width, dtype=dtype).requires_grad_(case["train"]) if case["residual"] else None
        if case["train"]:
            st["dout"] = randn(rows, width, dtype=dtype)
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _heads(x):
    """[B, L, H, D] -> [B, H, L, D] in 32 bits."""
    return x.detach().float().transpose(1, 2)


def _plain_attend(st):
    q = _heads(st["q"])
    k, v = (_heads(x) for x in (st["kv"].unbind(2) if st["packed"] else (st["k"], st["v"])))
    b, h, lq, d = q.shape
    hkv, lk = k.shape[1], k.shape[2]
    q = q.reshape(b, hkv, (h // hkv) * lq, d)  # the queries of the heads that share keys, side by side
    scale = 1.0 / math.sqrt(d)
    s = (q @ k.transpose(-1, -2)) * scale
    keep = None
    if st["key_lengths"] is not None:
        keep = torch.arange(lk, device=q.device) < st["key_lengths"][:, None]
    if st["key_mask"] is not None:
        keep = st["key_mask"]
    if keep is not None:
        s = s.masked_fill(~keep[:, None, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)  # a row without keys has no weights: its output is zero
    back = lambda x, heads, rows: x.reshape(b, heads, rows, d).transpose(1, 2).to(st["q"].dtype)  # noqa: E731
    o = p @ v
    if not st["train"]:
        return (back(o, h, lq),)
    do = _heads(st["dout"]).reshape(q.shape)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * scale
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    grads = (back(dk, hkv, lk), back(dv, hkv, lk))
    if st["packed"]:
        grads = (torch.stack(grads, dim=2),)
    return (back(o, h, lq), back(dq, h, lq), *grads)


def _plain_embed(st):
    w = st["weight"].detach()
    out = (w[st["token_ids"]].float() * st["scale"]).to(DTYPES[st["dtype"]])
    if not st["train"]:
        return (out,)
    dy = st["dout"].float() * st["scale"]
    if st["padding_idx"] is not None:
        dy = dy * (st["token_ids"] != st["padding_idx"])[:, None]
    dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32).index_add_(0, st["token_ids"], dy)
    return out, dw.to(w.dtype)


def _shift_right(z, n):
    """Logical right shift of 64-bit words held as signed integers."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _signed(c):
    return c - (1 << 64) if c >= 1 << 63 else c


def _plain_keep(seed, n, p):
    """The keep rule of the framework's dropout: element e is kept where the (e mod 4)-th 16 bits of
    splitmix64(seed ^ (e div 4) * 0xD1B54A32D192ED03) are at least p * 65536."""
    z = torch.arange((n + 3) // 4, device=seed.device) * _signed(0xD1B54A32D192ED03)
    z = (seed ^ z) + _signed(0x9E3779B97F4A7C15)
    z = (z ^ _shift_right(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shift_right(z, 27)) * _signed(0x94D049BB133111EB)
    z = z ^ _shift_right(z, 31)
    words = torch.stack((z & 0xFFFF, (z >> 16) & 0xFFFF, (z >> 32) & 0xFFFF, (z >> 48) & 0xFFFF), dim=1)
    return words.reshape(-1)[:n] >= round(p * 65536)


def _plain_dropout(st):
    x = st["x"].detach()
    factor = _plain_keep(st["seed"], x.numel(), st["p"]).reshape(x.shape) * (1.0 / (1.0 - st["p"]))
    y = x.float() * factor
    if st["add"] is not None:
        y = y + st["add"].detach().float()
    y = y.to(x.dtype)
    if not st["train"]:
        return (y,)
    dx = (st["dout"].float() * factor).to(x.dtype)
    return (y, dx) if st["add"] is None else (y, dx, st["dout"])


# ------------------------------------------------------------------------------------------ the framework's
def _package():
    if "diffusion-profiled_b200" not in sys.path:
        sys.path.insert(0, "diffusion-profiled_b200")
    import fp8_b200.cross_attention
    import fp8_b200.dropout
    import fp8_b200.embedding

    return fp8_b200


def _own_attend(st):
    attention = _package().cross_attention
    masks = {"key_lengths": st["key_lengths"], "key_mask": st["key_mask"]}
    if st["packed"]:
        inputs = (st["q"], st["kv"])
        o = attention.cross_attention_packed(*inputs, **masks)
    else:
        inputs = (st["q"], st["k"], st["v"])
        o = attention.cross_attention(*inputs, **masks)
    if not st["train"]:
        return (o,)
    return (o.detach(), *torch.autograd.grad(o, inputs, st["dout"]))


def _own_embed(st):
    out = _package().embedding.embed_tokens(st["token_ids"], st["weight"], scale=st["scale"],
                                            padding_idx=st["padding_idx"], dtype=DTYPES[st["dtype"]])
    if not st["train"]:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, (st["weight"],), st["dout"]))


def _own_dropout(st):
    drop = _package().dropout
    if st["add"] is None:
        inputs = (st["x"],)
        y = drop.dropout(st["x"], st["p"], st["seed"])
    else:
        inputs = (st["x"], st["add"])
        y = drop.dropout_add(st["x"], st["add"], st["p"], st["seed"])
    if not st["train"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, inputs, st["dout"]))


def run(state):
    forms = {"attend": (_plain_attend, _own_attend), "embed": (_plain_embed, _own_embed),
             "dropout": (_plain_dropout, _own_dropout)}
    return forms[state["op"]][1 if own else 0](state)


# ------------------------------------------------------------------------------------------ work and exact values
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "attend":
        b, lq, lk, h, hkv, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
        keys = {"none": lambda: b * lk, "lengths": lambda: sum(_lengths(case)), "mask": lambda: sum(_kept(case))}
        keys = keys[case["mask"]]()
        queries, states = b * lq * h * d * size, 2 * keys * hkv * d * size
        mask = b * lk if case["mask"] == "mask" else 4 * b if case["mask"] == "lengths" else 0
        if not case["train"]:
            return {"bytes": 2 * queries + states + mask, "flops": 4 * lq * keys * h * d}
        # forward: q, k, v in, o out; backward: q, k, v, o and its gradient in, three gradients out
        return {"bytes": 2 * queries + states + 4 * queries + states + 2 * b * lk * hkv * d * size + 2 * mask,
                "flops": 14 * lq * keys * h * d}
    if case["op"] == "embed":
        n, width, wsize = case["tokens"], case["width"], SIZE[case["wdtype"]]
        forward = 8 * n + min(n, case["vocab"]) * width * wsize + n * width * size
        if not case["train"]:
            return {"bytes": forward, "flops": n * width}
        return {"bytes": forward + 8 * n + n * width * size + case["vocab"] * width * wsize, "flops": 3 * n * width}
    n = case["rows"] * case["width"]
    forward = (3 if case["residual"] else 2) * n * size
    if not case["train"]:
        return {"bytes": forward, "flops": n}
    return {"bytes": forward + 2 * n * size, "flops": 2 * n}


def _exact_attend(case, st):
    """Softmax attention by its definition, one sequence and key head at a time, in 64 bits."""
    b, lq, lk, h, hkv, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
    group = h // hkv
    f64 = lambda x: x.detach().double()  # noqa: E731
    q = f64(st["q"])
    k, v = (f64(st["kv"][:, :, 0]), f64(st["kv"][:, :, 1])) if case["packed"] else (f64(st["k"]), f64(st["v"]))
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    for i in range(b):
        which = torch.arange(lk, device=q.device)
        if st["key_lengths"] is not None:
            which = which[: int(st["key_lengths"][i])]
        if st["key_mask"] is not None:
            which = which[st["key_mask"][i]]
        if not len(which):
            continue
        for head in range(h):
            shared = head // group
            ki, vi, qi = k[i, which, shared], v[i, which, shared], q[i, :, head]
            w = torch.softmax(qi @ ki.T / d**0.5, dim=-1)
            o[i, :, head] = w @ vi
            if case["train"]:
                g = f64(st["dout"])[i, :, head]
                gw = g @ vi.T
                gs = w * (gw - (g * o[i, :, head]).sum(-1, keepdim=True))
                dq[i, :, head] = gs @ ki / d**0.5
                dk[i, which, shared] += gs.T @ qi / d**0.5
                dv[i, which, shared] += w.T @ g
    if not case["train"]:
        return (o,)
    return (o, dq, torch.stack((dk, dv), 2)) if case["packed"] else (o, dq, dk, dv)


def _exact_embed(case, st):
    w = st["weight"].detach().double()
    out = torch.index_select(w, 0, st["token_ids"]) * st["scale"]
    if not case["train"]:
        return (out,)
    live = torch.ones_like(st["token_ids"], dtype=torch.bool)
    if st["padding_idx"] is not None:
        live = st["token_ids"] != st["padding_idx"]
    dw = torch.zeros_like(w)
    dw.index_put_((st["token_ids"][live],), st["dout"][live].double() * st["scale"], accumulate=True)
    return out, dw


def _exact_dropout(case, st):
    n = case["rows"] * case["width"]
    seed = np.uint64(int(st["seed"]) % 2**64)
    with np.errstate(over="ignore"):
        z = np.arange((n + 3) // 4, dtype=np.uint64) * np.uint64(0xD1B54A32D192ED03) ^ seed
        z += np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ z >> np.uint64(30)) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ z >> np.uint64(27)) * np.uint64(0x94D049BB133111EB)
        z ^= z >> np.uint64(31)
    kept = z.astype("<u8").view("<u2")[:n].astype(np.int64) >= round(case["p"] * 65536)
    keep = torch.from_numpy(kept).to(st["x"].device).reshape(case["rows"], case["width"])
    y = torch.where(keep, st["x"].detach().double() / (1 - case["p"]), 0.0)
    if st["add"] is not None:
        y = y + st["add"].detach().double()
    if not case["train"]:
        return (y,)
    dx = torch.where(keep, st["dout"].double() / (1 - case["p"]), 0.0)
    return (y, dx) if st["add"] is None else (y, dx, st["dout"].double())


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "embed": _exact_embed, "dropout": _exact_dropout}[case["op"]](case, st)
