"""Timed cases of the operators on a layer's hidden states: the token embedding
and its gradient, hidden dropout from a counter-based generator, the RMS norm
with the residual's addition, and the same with an output in 8 bits.

Each case is one call a user's program makes: a serving pass, or a training
step's forward and backward of the operator.  ``listed()`` names the cases,
``draw`` gives more of the same ranges, ``prepare`` builds what the program
holds before the call and ``run`` makes it, in elementary torch operations
(float32, rounded once at the end), or through this package's entry points
where ``own`` is set.  ``exact`` is the operator's definition in float64.

Sizes follow the repository's configurations (hidden 128, 768 and 1024,
vocabulary 128100, rows of 512 tokens, 4096 packed) and generic ones around
them, odd ones included.

Dropout's random numbers are a 64-bit seed: the value at row r (all leading
dimensions flattened) and column c is kept where 16 bits of
Philox4x32-10(counter = (c // 8, r & 0xffffffff, r >> 32, 0x68696464), key =
(seed & 0xffffffff, seed >> 32)) are at least t = round(65536 p): of word
(c % 8) // 2 the low half for even c, the high half for odd c.  A kept value is
scaled by 65536 / (65536 - t).
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4, "none": 0}
EPS = 1e-6
DOMAIN = 0x68696464  # the counter's last word
FP8_MAX = 448.0  # the largest value of float8_e4m3fn
MOST_TOKENS, MOST_VALUES = 131072, 1 << 26  # of a drawn case, as the largest listed ones


# ---------------------------------------------------------------------------
# the cases


def _embed(name, batch, length, hidden, vocab, weight, out, pad, train):
    """pad: the share of padded positions (id 0, the padding index)."""
    return {"name": name, "op": "embed", "batch": batch, "length": length, "hidden": hidden, "vocab": vocab,
            "weight": weight, "out": out, "pad": pad, "train": train}


def _dropout(name, batch, length, hidden, dtype, res, bias, p, train=True):
    """res: the residual's type or "none"; bias: with a float32 bias."""
    return {"name": name, "op": "dropout", "batch": batch, "length": length, "hidden": hidden, "dtype": dtype,
            "res": res, "bias": bias, "p": p, "train": train}


def _rms(name, batch, length, hidden, dtype, res, param, bias, p, train):
    """param: the type of the norm's weight and of the bias."""
    return {"name": name, "op": "rms", "batch": batch, "length": length, "hidden": hidden, "dtype": dtype, "res": res,
            "param": param, "bias": bias, "p": p, "train": train}


def _rms_fp8(name, batch, length, hidden, dtype, res, group):
    """group: columns that share a scale, 0 for one scale a row."""
    return {"name": name, "op": "rms_fp8", "batch": batch, "length": length, "hidden": hidden, "dtype": dtype,
            "res": res, "group": group}


def listed():
    return [
        # serving: the lookup of one new token for each of eight requests
        _embed("embed_tokens", 8, 1, 768, 128100, "bf16", "bf16", 0.0, False),
        # a training step of the base encoder's embedding under mixed precision: float32 master weights
        _embed("embed_train_base", 16, 512, 768, 128100, "fp32", "fp32", 0.25, True),
        # a ragged batch of a small model with an odd width, weights in bf16
        _embed("embed_train_odd", 7, 389, 513, 50021, "bf16", "bf16", 0.4, True),
        # packed long rows of the large encoder, weights held in bf16
        _embed("embed_train_packed", 32, 4096, 1024, 128100, "bf16", "bf16", 0.0, True),
        # a smoke-sized training step of a sublayer's end
        _dropout("dropout_small", 2, 128, 128, "fp32", "fp32", True, 0.1),
        # the base encoder's sublayer end: dropout of the dense output with its bias, plus the residual
        _dropout("dropout_base", 32, 512, 768, "bf16", "bf16", True, 0.1),
        # embeddings of the large encoder's packed rows, plain dropout; odd width
        _dropout("dropout_packed_odd", 16, 4096, 1023, "bf16", "none", False, 0.15),
        # serving: the norm of one token, with the residual stream in float32
        _rms("rms_token", 1, 1, 1024, "bf16", "fp32", "fp32", False, 0.0, False),
        # a training step of a base-sized pre-norm sublayer, with its bias and hidden dropout
        _rms("rms_train_base", 32, 512, 768, "bf16", "bf16", "bf16", True, 0.1, True),
        # a wide model under mixed precision: float32 residual stream and parameters
        _rms("rms_train_wide", 4, 4096, 4096, "bf16", "fp32", "fp32", False, 0.0, True),
        # serving in 8 bits: a few tokens of a wide model, a scale for each 128 columns
        _rms_fp8("rms_fp8_tokens", 4, 1, 4096, "bf16", "bf16", 128),
        # serving in 8 bits: a ragged prompt batch of the large encoder, one scale a row
        _rms_fp8("rms_fp8_prompt", 13, 767, 1024, "bf16", "bf16", 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows(rng, most):
    """batch and length of at most ``most`` rows, from a single token to packed rows."""
    rows = _log(rng, 1, most)
    batch = _log(rng, 1, min(64, rows))
    return batch, max(1, rows // batch)


def draw(rng: random.Random):
    op = rng.choice(("embed", "dropout", "rms", "rms_fp8"))
    dtype, train = rng.choice(("bf16", "fp32")), rng.random() < 0.7
    res = rng.choice(("none", dtype, "fp32"))
    if op == "embed":
        batch, length = _rows(rng, MOST_TOKENS)
        case = _embed("", batch, length, _log(rng, 33, 1024), _log(rng, 1000, 128100), dtype,
                      rng.choice((dtype, "bf16")), rng.choice((0.0, rng.uniform(0.05, 0.6))), train)
        if dtype == "fp32":  # no more bytes than the largest listed case
            case["length"] = max(1, length // 2)
            case["vocab"] = max(1000, case["vocab"] // 2)
    elif op == "dropout":
        hidden = _log(rng, 33, 4096)
        batch, length = _rows(rng, min(MOST_TOKENS, MOST_VALUES // (4 * hidden)))
        case = _dropout("", batch, length, hidden, dtype, res, rng.random() < 0.5, rng.choice((0.1, rng.uniform(0.02, 0.5))), train)
    elif op == "rms":
        hidden = _log(rng, 33, 8192)
        batch, length = _rows(rng, min(MOST_TOKENS, MOST_VALUES // (2 * hidden)))
        case = _rms("", batch, length, hidden, dtype, res, rng.choice((dtype, "fp32")), rng.random() < 0.5,
                    rng.choice((0.0, 0.0, 0.1, rng.uniform(0.02, 0.3))) if train else 0.0, train)
    else:
        group = rng.choice((0, 32, 64, 128))
        hidden = _log(rng, 33, 8192)
        if group:
            hidden = max(group, hidden // group * group)
        batch, length = _rows(rng, min(MOST_TOKENS, MOST_VALUES // (2 * hidden)))
        case = _rms_fp8("", batch, length, hidden, dtype, res, group)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# what a program holds before the call


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    B, L, C = case["batch"], case["length"], case["hidden"]
    s = SimpleNamespace(case=dict(case), C=C, train=case.get("train", False))
    leaf = lambda t: t.requires_grad_(s.train)  # noqa: E731
    if case["op"] == "embed":
        V = case["vocab"]
        s.weight = leaf((randn(V, C) * 0.02).to(TYPES[case["weight"]]))
        # token frequencies fall as 1 / rank
        u = torch.rand((B, L), generator=g, device=DEV, dtype=torch.float64)
        s.ids = torch.exp(u * math.log(V)).long().clamp_(1, V - 1)
        if case["pad"]:  # every row ends in padding, by case["pad"] on average
            lens = 1 + (torch.rand((B, 1), generator=g, device=DEV) * 2 * (1 - case["pad"])).clamp(max=1.0) * (L - 1)
            s.ids.masked_fill_(torch.arange(L, device=DEV)[None, :] >= lens, 0)
        s.out_dtype = TYPES[case["out"]]
        s.scale = math.sqrt(C)
        if s.train:
            s.dy = randn(B, L, C).to(s.out_dtype)
        return s
    dtype = TYPES[case["dtype"]]
    s.x = leaf(randn(B, L, C).to(dtype))
    s.res = leaf(randn(B, L, C).to(TYPES[case["res"]])) if case["res"] != "none" else None
    s.z_dtype = dtype if s.res is None else torch.promote_types(dtype, s.res.dtype)
    s.seed = torch.randint(0, 1 << 62, (1,), generator=torch.Generator().manual_seed(int(seed)), dtype=torch.int64)
    param = TYPES[case.get("param", "fp32")]
    s.bias = leaf((randn(C) * 0.5).to(param)) if case.get("bias") else None
    if case["op"] == "dropout":
        if s.train:
            s.dy = randn(B, L, C).to(s.z_dtype)
        return s
    s.weight = leaf((1.0 + 0.2 * randn(C)).to(param if case["op"] == "rms" else torch.float32))
    if s.train:
        s.dy = randn(B, L, C).to(s.z_dtype)
        s.dz = randn(B, L, C).to(s.z_dtype)
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    c = s.case
    if c["op"] == "embed":
        return _own_embed(s) if own else _plain_embed(s)
    if c["op"] == "dropout":
        return _own_dropout(s) if own else _plain_dropout(s)
    if c["op"] == "rms":
        return _own_rms(s) if own else _plain_rms(s)
    return _own_rms_fp8(s) if own else _plain_rms_fp8(s)


def _own_embed(s):
    from deberta_amd import fused_embedding

    y = fused_embedding(s.ids, s.weight, padding_idx=0, scale=s.scale, out_dtype=s.out_dtype)
    if not s.train:
        return (y,)
    return (y, *torch.autograd.grad(y, (s.weight,), s.dy))


def _own_dropout(s):
    from deberta_amd import fused_dropout

    y = fused_dropout(s.x, s.case["p"], bias=s.bias, res=s.res, seed=s.seed)
    if not s.train:
        return (y,)
    return (y, *torch.autograd.grad(y, [t for t in (s.x, s.bias) if t is not None], s.dy))


def _own_rms(s):
    from deberta_amd import fused_add_rms_norm

    p = s.case["p"]
    y, z = fused_add_rms_norm(s.x, s.weight, EPS, bias=s.bias, res=s.res, dropout_p=p, seed=s.seed if p else None,
                              out_dtype=s.z_dtype)
    if not s.train:
        return (y, z)
    leaves = [t for t in (s.x, s.bias, s.res, s.weight) if t is not None]
    return (y, z, *torch.autograd.grad((y, z), leaves, (s.dy, s.dz)))


def _own_rms_fp8(s):
    from deberta_amd import fused_add_rms_norm_fp8

    return fused_add_rms_norm_fp8(s.x, s.weight, EPS, bias=s.bias, res=s.res, group_size=s.case["group"] or None)


@torch.no_grad()
def _plain_embed(s):
    y = (s.weight[s.ids].float() * s.scale).to(s.out_dtype)
    if not s.train:
        return (y,)
    dy = s.dy.float() * s.scale * (s.ids != 0).unsqueeze(-1)
    dw = torch.zeros(s.weight.shape, device=DEV).index_add_(0, s.ids.reshape(-1), dy.reshape(-1, s.C))
    return (y, dw.to(s.weight.dtype))


def _threshold(p):
    return int(round(p * 65536.0))


def _plain_scale(s, p):
    """The factor of every value: 65536 / (65536 - t) where it is kept, else 0."""
    t = _threshold(p)
    rows, groups = s.x.numel() // s.C, -(-s.C // 8)
    seed = s.seed.item()
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    low = 0xFFFFFFFF
    r = torch.arange(rows, device=DEV)
    shape = (rows, groups)
    c0 = torch.arange(groups, device=DEV)[None, :].expand(shape)
    c1, c2 = (r & low)[:, None].expand(shape), (r >> 32)[:, None].expand(shape)
    c3 = torch.full_like(c2, DOMAIN)
    for _ in range(10):  # products wrap in 64 bits: their words are right all the same
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), -1)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1)
    keep = halves.reshape(rows, groups * 8)[:, : s.C] >= t
    return (keep * (65536.0 / (65536 - t))).float().view(s.x.shape)


def _plain_sum(s, factor):
    """x + bias, times the factor, plus the residual, in float32."""
    z = s.x.float()
    if s.bias is not None:
        z = z + s.bias.float()
    if factor is not None:
        z = z * factor
    return z if s.res is None else z + s.res.float()


@torch.no_grad()
def _plain_dropout(s):
    factor = _plain_scale(s, s.case["p"])
    y = _plain_sum(s, factor).to(s.z_dtype)
    if not s.train:
        return (y,)
    dx = s.dy.float() * factor
    out = [y, dx.to(s.x.dtype)]
    if s.bias is not None:
        out.append(dx.reshape(-1, s.C).sum(0).to(s.bias.dtype))
    return tuple(out)


@torch.no_grad()
def _plain_rms(s):
    factor = _plain_scale(s, s.case["p"]) if s.case["p"] else None
    z = _plain_sum(s, factor)
    w = s.weight.float()
    r = 1.0 / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS)
    out = [(z * r * w).to(s.z_dtype), z.to(s.z_dtype)]
    if not s.train:
        return tuple(out)
    dy = s.dy.float()
    g = dy * w
    dz = r * (g - z * (r * r * (g * z).mean(-1, keepdim=True))) + s.dz.float()
    dx = dz if factor is None else dz * factor
    out.append(dx.to(s.x.dtype))
    if s.bias is not None:
        out.append(dx.reshape(-1, s.C).sum(0).to(s.bias.dtype))
    if s.res is not None:
        out.append(dz.to(s.res.dtype))
    out.append((dy * z * r).reshape(-1, s.C).sum(0).to(s.weight.dtype))
    return tuple(out)


@torch.no_grad()
def _plain_rms_fp8(s):
    z = _plain_sum(s, None)
    y = z / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS) * s.weight.float()
    group = s.case["group"] or s.C
    y = y.unflatten(-1, (s.C // group, group))
    scale = y.abs().amax(-1, keepdim=True) / FP8_MAX
    scale = torch.where(scale < 2.0**-126, 1.0, scale)
    q = (y / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).flatten(-2)
    return (q, scale.squeeze(-1), z.to(s.z_dtype))


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    rows, C = case["batch"] * case["length"], case["hidden"]
    n = rows * C
    if case["op"] == "embed":
        V, w, o = case["vocab"], BYTES[case["weight"]], BYTES[case["out"]]
        # the frequencies fall as 1 / rank: the number of distinct tokens, expected
        tokens = rows * (1.0 - case["pad"])
        ranks = [int(V ** (i / 256)) for i in range(257)]
        distinct = 1.0
        for lo, hi in zip(ranks, ranks[1:]):
            if hi > lo:
                share = math.log(hi / lo) / math.log(V) / (hi - lo)
                distinct += (hi - lo) * -math.expm1(-tokens * share)
        b = rows * 8 + distinct * C * w + n * o
        if case["train"]:
            b += n * o + V * C * w
        return {"bytes": b, "flops": n * (2.0 if case["train"] else 1.0)}
    x, res = BYTES[case["dtype"]], BYTES[case["res"]]
    z = max(x, res)
    # Philox4x32-10: ten rounds of two products and eight more operations for eight values
    random_ops = 12.5 * n if case.get("p") else 0.0
    if case["op"] == "dropout":
        b, f = n * (x + res + z), 3.0 * n + random_ops
        if case["train"]:
            b, f = b + n * (z + x), 2 * f
        return {"bytes": b, "flops": f}
    if case["op"] == "rms":
        b, f = n * (x + res + 2 * z), 6.0 * n + random_ops
        if case["train"]:
            b, f = b + n * (2 * z + x + res + x + res), 3 * f
        return {"bytes": b + 8 * C, "flops": f}
    return {"bytes": n * (x + res + z + 1) + 4 * rows * (C // case["group"] if case["group"] else 1) + 4 * C, "flops": 9.0 * n}


# ---------------------------------------------------------------------------
# the definitions, in float64


def _exact_keep(seed, rows, C, t):
    """Which values are kept, row by row, in numpy's unsigned integers."""
    m32 = np.uint64(0xFFFFFFFF)
    kept = np.empty((rows, -(-C // 8) * 8), dtype=bool)
    lanes = np.arange(kept.shape[1] // 8, dtype=np.uint64)
    step = max(1, (1 << 20) // len(lanes))
    for lo in range(0, rows, step):
        r = np.arange(lo, min(rows, lo + step), dtype=np.uint64)
        ctr = [np.broadcast_to(v, (len(r), len(lanes))) for v in
               (lanes[None, :], (r & m32)[:, None], (r >> np.uint64(32))[:, None], np.uint64(DOMAIN))]
        key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), b & m32,
                   (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), a & m32]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for u in range(8):
            kept[lo : lo + len(r), u::8] = (ctr[u // 2] >> np.uint64(16 * (u % 2)) & np.uint64(0xFFFF)) >= t
    return torch.from_numpy(kept[:, :C])


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    C = s.C
    if case["op"] == "embed":
        flat = s.ids.reshape(-1)
        out = [s.weight.double().index_select(0, flat).mul_(s.scale).view(*s.ids.shape, C)]
        if s.train:
            # prefix sums over the tokens in order, a block of columns at a time
            order = torch.argsort(flat, stable=True)
            counts = torch.bincount(flat, minlength=case["vocab"])
            ends = counts.cumsum(0)
            dw = torch.zeros(case["vocab"], C, dtype=torch.float64, device=DEV)
            dy = s.dy.reshape(-1, C)
            for lo in range(0, C, 128):
                sums = torch.nn.functional.pad(dy[:, lo : lo + 128].double()[order].cumsum(0), (0, 0, 1, 0))
                dw[:, lo : lo + 128] = (sums[ends] - sums[ends - counts]) * s.scale
            dw[0] = 0.0
            out.append(dw)
        return tuple(out)
    rows = s.x.numel() // C
    kept = 1.0
    t = _threshold(case.get("p", 0.0))
    if t:
        kept = _exact_keep(int(s.seed), rows, C, t).to(DEV).double().mul_(65536.0 / (65536 - t))
    z = s.x.double().view(rows, C)
    if s.bias is not None:
        z = z + s.bias.double()
    z = z * kept
    if s.res is not None:
        z = z + s.res.double().view(rows, C)
    shaped = lambda v: v.view(s.x.shape)  # noqa: E731
    if case["op"] == "dropout":
        out = [shaped(z)]
        if s.train:
            dx = s.dy.double().view(rows, C) * kept
            out.append(shaped(dx))
            if s.bias is not None:
                out.append(dx.sum(0))
        return tuple(out)
    inv = (z.square().sum(1, keepdim=True) / C + EPS).rsqrt()
    w = s.weight.double()
    y = z * inv * w
    if case["op"] == "rms":
        out = [shaped(y), shaped(z)]
        if s.train:
            dy = s.dy.double().view(rows, C)
            normed = z * inv
            g = dy * w
            dz = inv * (g - normed * ((g * normed).sum(1, keepdim=True) / C)) + s.dz.double().view(rows, C)
            dx = dz * kept
            out.append(shaped(dx))
            if s.bias is not None:
                out.append(dx.sum(0))
            if s.res is not None:
                out.append(shaped(dz))
            out.append((dy * normed).sum(0))
        return tuple(out)
    # in 8 bits: the values before their rounding, in units of the scale
    group = case["group"] or C
    y = y.view(rows, C // group, group)
    scale = y.abs().max(2, keepdim=True).values / FP8_MAX
    q = y / scale
    return (shaped(q), scale.view(*s.x.shape[:-1], C // group), shaped(z))
