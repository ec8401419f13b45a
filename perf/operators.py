"""What the operators of the package's training side cost: dropout from a counter-based generator, the relative position
encoding of pairs, and attention with a sliding window.

A pair tensor has some dozens to some 1500 tokens a side and 128 channels; the single representation 384 channels in 16
heads of 24; sequence-local attention runs over atoms (4 heads of 32, about eight atoms a token, several samples of one
structure at once) and over long chains.  A training step returns what it gives the optimiser: the gradients.

With ``own`` false, ``run`` is elementary tensor operations in 32 bits (the generator's integers in 64); with ``own``
true it makes the calls that a user of the package makes.  Both take the same state.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
C_Z, C_S = 128, 384
R_MAX, S_MAX = 32, 2                                     # the encoding's clipping distances


def listed():
    return [
        # Element-wise dropout of the single representation's update, one crop of 384 tokens: latency.
        {"name": "dropout_single_384", "op": "dropout", "shape": f"384,{C_S}", "shared": 0, "p": 0.1, "dtype": "bf16"},
        # Row-shared dropout of a triangle update in a training crop, fp32 residual stream.
        {"name": "dropout_row_512", "op": "dropout", "shape": f"512,512,{C_Z}", "shared": -3, "p": 0.25, "dtype": "fp32"},
        # Element-wise dropout of a whole pair tensor: as much generator work as there is, per byte.
        {"name": "dropout_pair_768", "op": "dropout", "shape": f"768,768,{C_Z}", "shared": 0, "p": 0.15, "dtype": "bf16"},
        # The encoding of a short chain: forward alone, latency.
        {"name": "relpos_97", "op": "relpos", "n": 97, "chains": 1, "dtype": "fp32", "train": False},
        # A training crop: the encoding and the gradient of its weight.
        {"name": "relpos_train_384", "op": "relpos", "n": 384, "chains": 4, "dtype": "fp32", "train": True},
        # The benchmark's largest complex in training, many chains, odd length.
        {"name": "relpos_train_1501", "op": "relpos", "n": 1501, "chains": 11, "dtype": "bf16", "train": True},
        # One short chain through local attention in inference.
        {"name": "attn_short_97", "op": "attn", "batch": 1, "n": 97, "heads": 4, "kv_heads": 4, "d": 32, "left": 64, "right": 63,
         "sinks": 0, "r_max": 0, "pad": 0, "dtype": "bf16", "train": False},
        # Atoms of five samples of a crop in training: 128 keys around an atom, a learned bias by offset, padded at the end.
        {"name": "attn_atoms_train", "op": "attn", "batch": 5, "n": 3987, "heads": 4, "kv_heads": 4, "d": 32, "left": 64,
         "right": 63, "sinks": 0, "r_max": 32, "pad": 75, "dtype": "bf16", "train": True},
        # The single representation's heads of 24 over a long complex, padded in front, so that rows there see nothing.
        {"name": "attn_single_train", "op": "attn", "batch": 2, "n": 1237, "heads": 16, "kv_heads": 16, "d": 24, "left": 200,
         "right": 200, "sinks": 5, "r_max": 32, "pad": -37, "dtype": "fp16", "train": True},
        # A causal window over a long sequence, heads of k and v shared by four, first tokens kept visible: training.
        {"name": "attn_causal_train", "op": "attn", "batch": 1, "n": 8192, "heads": 16, "kv_heads": 4, "d": 64, "left": 1023,
         "right": 0, "sinks": 4, "r_max": 128, "pad": 0, "dtype": "bf16", "train": True},
        # The longest sequence, large heads, forward alone.
        {"name": "attn_long_16384", "op": "attn", "batch": 1, "n": 16384, "heads": 8, "kv_heads": 2, "d": 128, "left": 2047,
         "right": 0, "sinks": 16, "r_max": 0, "pad": 0, "dtype": "bf16", "train": False},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "relpos", "attn", "attn"])
    if op == "dropout":
        p = rng.choice([0.05, 0.1, 0.15, 0.25, 0.5])
        if rng.random() < 0.3:
            shape, shared = f"{_log(rng, 1, 16384)},{rng.choice([C_S, 129, 768])}", 0
        else:
            n = _log(rng, 16, 720)
            shape, shared = f"{n},{n},{C_Z}", rng.choice([0, -2, -3])
        return {"op": op, "shape": shape, "shared": shared, "p": p, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "relpos":
        n = _log(rng, 16, 1400)
        return {"op": op, "n": n, "chains": rng.randint(1, max(1, min(12, n // 8))), "dtype": rng.choice(["fp32", "bf16"]),
                "train": rng.random() < 0.6}
    heads, kv_heads, d = rng.choice([(4, 4, 32), (16, 16, 24), (16, 16, 48), (8, 8, 64), (8, 2, 128), (16, 4, 64), (6, 2, 40)])
    n = _log(rng, 16, 8192)
    batch = max(1, min(_log(rng, 1, 8), int(9e8 / (heads * n * n))))
    left = _log(rng, 1, 2048)
    right = rng.choice([0, 0, left, _log(rng, 1, 512)])
    return {"op": op, "batch": batch, "n": n, "heads": heads, "kv_heads": kv_heads, "d": d, "left": left, "right": right,
            "sinks": rng.choice([0, 1, 4, 37]), "r_max": rng.choice([0, 8, 32, 128]), "pad": rng.choice([0, n // 11, -(n // 13)]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "train": rng.random() < 0.6}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _features(n, chains, g):
    """Chains one behind the other, some of them copies of one entity; residues numbered from 1 with a break, a tail of
    atoms that share their residue number (a ligand)."""
    cpu = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=g, device="cuda")))
    cuts = torch.randperm(n - 1, generator=cpu)[: chains - 1].add(1).sort().values if chains > 1 else torch.zeros(0, dtype=torch.long)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), cuts])
    asym = torch.zeros(n, dtype=torch.long)
    asym[starts[1:]] = 1
    asym = asym.cumsum(0)
    place = torch.arange(n) - starts[asym]
    entity = asym // 2
    residue = place + 1 + 7 * (place > 40).long()
    tail = (asym == asym[-1]) & (torch.arange(n) >= n - max(1, n // 10))
    residue[tail] = int(residue[tail][0])
    feats = {"asym_id": asym, "residue_index": residue, "entity_id": entity, "token_index": torch.arange(n), "sym_id": asym % 2}
    return {k: v.cuda() for k, v in feats.items()}


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "dropout":
        shape = [int(x) for x in case["shape"].split(",")]
        s["residual"] = _randn(g, *shape, dtype=dtype).requires_grad_()
        s["x"] = _randn(g, *shape, dtype=dtype).requires_grad_()
        s["grad"] = _randn(g, *shape, dtype=dtype)
        s["seed"], s["offset"] = 1234567890123 + 97 * seed, seed % 1000   # what the program's own counter stands at
    elif case["op"] == "relpos":
        s["features"] = _features(case["n"], case["chains"], g)
        s["weight"] = _randn(g, C_Z, 4 * R_MAX + 2 * S_MAX + 7, std=0.1).requires_grad_(case["train"])
        if case["train"]:
            s["grad"] = _randn(g, case["n"], case["n"], C_Z, dtype=dtype)
    else:
        b, n, h, hk, d = (case[k] for k in ("batch", "n", "heads", "kv_heads", "d"))
        # one projection gives q, k and v of all heads: the heads are views into its rows
        qkv = _randn(g, b, n, h + 2 * hk, d, dtype=dtype)
        q, k, v = (t.transpose(1, 2) for t in qkv.split([h, hk, hk], dim=2))
        s["q"], s["k"], s["v"] = (t.detach().requires_grad_(case["train"]) for t in (q, k, v))
        # the learned bias in the type of the projections, as a layer cast to 16 bits has it
        s["rel_bias"] = _randn(g, h, 2 * case["r_max"] + 1, dtype=dtype, std=0.5).requires_grad_(case["train"]) if case["r_max"] else None
        s["mask"] = None
        if case["pad"]:
            s["mask"] = torch.ones(b, n, dtype=torch.bool, device="cuda")
            for i in range(b):                            # each sample has its own length
                pad = max(1, abs(case["pad"]) * (i + 1) // b)
                if case["pad"] > 0:
                    s["mask"][i, n - pad:] = False
                else:
                    s["mask"][i, :pad] = False
        if case["train"]:
            s["grad"] = _randn(g, b, n, h, d, dtype=dtype).transpose(1, 2)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"dropout": _plain_dropout, "relpos": _plain_relpos, "attn": _plain_attn}[s["op"]](s)


def _own(s):
    import protenix_b200 as px

    if s["op"] == "dropout":
        out = px.dropout_add(s["residual"], s["x"], s["p"], s["seed"], offset=s["offset"], shared_dim=s["shared"] or None)
        return out.detach(), *torch.autograd.grad(out, (s["residual"], s["x"]), s["grad"])
    if s["op"] == "relpos":
        z = px.relative_position_encoding(s["weight"], **s["features"], r_max=R_MAX, s_max=S_MAX, dtype=DTYPES[s["dtype"]])
        return (z.detach(), *torch.autograd.grad(z, (s["weight"],), s["grad"])) if s["train"] else z
    o = px.window_attention(s["q"], s["k"], s["v"], (s["left"], s["right"]), sinks=s["sinks"], rel_bias=s["rel_bias"], mask=s["mask"])
    if not s["train"]:
        return o
    leaves = [t for t in (s["q"], s["k"], s["v"], s["rel_bias"]) if t is not None]
    return o.detach(), *torch.autograd.grad(o, leaves, s["grad"])


LOW = 0xFFFFFFFF


def _philox(c, key):
    """Ten rounds of Philox4x32 (Salmon et al., 2011) on four int64 tensors that hold 32 bits each."""
    k0, k1 = key
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57     # products wrap in 64 bits, which keeps every bit of them
        c = [(b >> 32 & LOW) ^ c[1] ^ k0, b & LOW, (a >> 32 & LOW) ^ c[3] ^ k1, a & LOW]
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return c


def _plain_dropout(s):
    x, p = s["x"], s["p"]
    shape = list(x.shape)
    if s["shared"]:
        shape[s["shared"]] = 1
    n = math.prod(shape)
    block = torch.arange((n + 3) // 4, device=x.device)
    fixed = [torch.full_like(block, s["offset"] >> sh & LOW) for sh in (0, 32)]
    words = torch.stack(_philox([block & LOW, block >> 32, *fixed], (s["seed"] & LOW, s["seed"] >> 32 & LOW)), dim=1)
    keep = (words.flatten()[:n] >= round(p * 2 ** 32)).view(shape)
    scale = 1.0 / (1.0 - p)
    zero = torch.zeros((), device=x.device)
    out = s["residual"].float() + torch.where(keep, x.float() * scale, zero)
    dx = torch.where(keep, s["grad"].float() * scale, zero)
    return out.to(x.dtype), s["grad"], dx.to(x.dtype)


def _buckets(f):
    """The three bucket numbers and the same-entity flag of every pair."""
    d = {k: v[:, None] - v[None, :] for k, v in f.items()}
    chain, entity = d["asym_id"] == 0, d["entity_id"] == 0
    pos = torch.where(chain, (d["residue_index"] + R_MAX).clamp(0, 2 * R_MAX), 2 * R_MAX + 1)
    tok = torch.where(chain & (d["residue_index"] == 0), (d["token_index"] + R_MAX).clamp(0, 2 * R_MAX), 2 * R_MAX + 1)
    sym = torch.where(entity, (d["sym_id"] + S_MAX).clamp(0, 2 * S_MAX), 2 * S_MAX + 1)
    return pos, tok, sym, entity


def _plain_relpos(s):
    pos, tok, sym, entity = _buckets(s["features"])
    w = s["weight"].float().t().contiguous()            # [buckets, c]
    m = 2 * R_MAX + 2
    at = (pos, tok + m, sym + 2 * m + 1)
    z = w[at[0]] + w[at[1]] + entity[..., None] * w[2 * m] + w[at[2]]
    z = z.to(DTYPES[s["dtype"]])
    if not s["train"]:
        return z
    dz = s["grad"].reshape(-1, C_Z).to(torch.float64)   # sums over up to some millions of pairs
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    dw.index_add_(0, at[0].flatten(), dz).index_add_(0, at[1].flatten(), dz).index_add_(0, at[2].flatten(), dz)
    dw[2 * m] = (dz * entity.flatten()[:, None]).sum(0)
    return z, dw.t().float().contiguous()


def _visible(s, rows, cols):
    """[.., N, N] truth values: which keys a query sees."""
    seen = (cols <= rows + s["right"]) & ((cols >= rows - s["left"]) | (cols < s["sinks"]))
    return seen if s["mask"] is None else seen & s["mask"][:, None, None, :]


def _plain_attn(s):
    q, k, v = (s[x].float() for x in "qkv")
    group = s["heads"] // s["kv_heads"]
    kf, vf = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    n, scale = s["n"], s["d"] ** -0.5
    i = torch.arange(n, device=q.device)
    logits = (q @ kf.transpose(-1, -2)).mul_(scale)
    bucket = None
    if s["rel_bias"] is not None:
        bucket = (i[None, :] - i[:, None]).clamp_(-s["r_max"], s["r_max"]).add_(s["r_max"])
        logits += s["rel_bias"].float()[:, bucket]
    logits.masked_fill_(~_visible(s, i[:, None], i[None, :]), -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min_(-3.0e38)              # a row that sees nothing has no largest logit
    p = logits.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp_min_(1e-37)
    o = p @ vf
    if not s["train"]:
        return o.to(s["q"].dtype)
    do = s["grad"].float()
    shared = lambda t: t.unflatten(1, (s["kv_heads"], group)).sum(2)  # noqa: E731
    dv = shared(p.transpose(-1, -2) @ do)
    ds = (do @ vf.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ kf).mul_(scale)
    dk = shared(ds.transpose(-1, -2) @ q).mul_(scale)
    out = [o.to(s["q"].dtype)] + [t.to(s["q"].dtype) for t in (dq, dk, dv)]
    if bucket is not None:
        ds = ds.sum(0)                                   # [heads, N, N]; rows shifted so that an offset is a column
        skewed = torch.nn.functional.pad(ds.flip(-1), (0, n)).flatten(1)[:, : n * (2 * n - 1)].view(-1, n, 2 * n - 1)
        by_offset = skewed.sum(1, dtype=torch.float64)   # column c: j - i = n - 1 - c
        at = torch.arange(n - 1, -n, -1, device=q.device).clamp_(-s["r_max"], s["r_max"]) + s["r_max"]
        db = torch.zeros(s["heads"], 2 * s["r_max"] + 1, dtype=torch.float64, device=q.device)
        out.append(db.index_add_(1, at, by_offset).to(s["q"].dtype))
    return tuple(out)


# ---- work and exact values -------------------------------------------------------------------------------------------
def _pairs(case):
    """Visible pairs of one head and sample, without its padding."""
    i = np.arange(case["n"], dtype=np.int64)
    low, high = np.maximum(i - case["left"], 0), np.minimum(i + case["right"], case["n"] - 1)
    return int((high - low + 1 + np.minimum(np.minimum(case["sinks"], low), high + 1)).sum())


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = math.prod(int(x) for x in case["shape"].split(","))
        return {"bytes": 5 * n * size, "flops": 3 * n}
    if case["op"] == "relpos":
        n = case["n"] ** 2 * C_Z
        table = C_Z * (4 * R_MAX + 2 * S_MAX + 7) * 4
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (n * size + table) + 5 * 8 * case["n"], "flops": passes * 3 * n}
    rows = case["batch"] * case["n"] * case["d"] * size
    pairs = case["batch"] * case["heads"] * _pairs(case)
    bytes_, flops = rows * 2 * (case["heads"] + case["kv_heads"]), 4 * case["d"] * pairs
    if case["train"]:
        bytes_, flops = bytes_ + rows * (4 * case["heads"] + 4 * case["kv_heads"]), flops + 10 * case["d"] * pairs
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"dropout": _exact_dropout, "relpos": _exact_relpos, "attn": _exact_attn}[case["op"]](s)


def _exact_dropout(s):
    shape = list(s["x"].shape)
    if s["shared"]:
        shape[s["shared"]] = 1
    n = int(np.prod(shape))
    u32, sh = np.uint64(LOW), np.uint64(32)
    at = np.arange(-(-n // 4), dtype=np.uint64)
    x0, x1 = at & u32, at >> sh
    x2, x3 = np.full_like(at, s["offset"] & LOW), np.full_like(at, s["offset"] >> 32)
    for r in range(10):
        k0, k1 = (np.uint64((s["seed"] >> z & LOW) + r * w & LOW) for z, w in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        lo, hi = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
        x0, x1, x2, x3 = hi >> sh ^ x1 ^ k0, hi & u32, lo >> sh ^ x3 ^ k1, lo & u32
    drop = np.stack([x0, x1, x2, x3], -1).reshape(-1)[:n] < np.uint64(round(s["p"] * 2 ** 32))
    m = torch.from_numpy(~drop).cuda().view(shape).double() / (1.0 - s["p"])
    return s["residual"].double() + s["x"].double() * m, s["grad"].double(), s["grad"].double() * m


def _exact_relpos(s):
    """The encoding as a linear map of one-hot vectors, a block of rows at a time."""
    f, w = s["features"], s["weight"].double()
    hot = torch.nn.functional.one_hot
    z, dw = [], torch.zeros_like(w)
    for i in range(0, s["n"], 64):
        same = {k: v[i:i + 64, None] == v[None] for k, v in f.items()}
        diff = {k: v[i:i + 64, None] - v[None] for k, v in f.items()}
        far = lambda d, r, ok: torch.where(ok, d.clamp(-r, r) + r, 2 * r + 1)  # noqa: E731
        one = torch.cat([
            hot(far(diff["residue_index"], R_MAX, same["asym_id"]), 2 * R_MAX + 2),
            hot(far(diff["token_index"], R_MAX, same["asym_id"] & same["residue_index"]), 2 * R_MAX + 2),
            same["entity_id"][..., None].long(), hot(far(diff["sym_id"], S_MAX, same["entity_id"]), 2 * S_MAX + 2)], -1).double()
        z.append(one @ w.t())
        if s["train"]:
            dw += s["grad"][i:i + 64].double().flatten(0, 1).t() @ one.flatten(0, 1)
    z = torch.cat(z)
    return (z, dw) if s["train"] else z


def _exact_attn(s):
    """One head of one sample at a time."""
    b, h, n, r = s["batch"], s["heads"], s["n"], s["r_max"]
    group, scale = h // s["kv_heads"], 1.0 / math.sqrt(s["d"])
    far = torch.arange(n, device="cuda")[None, :] - torch.arange(n, device="cuda")[:, None]         # j - i
    window = (far <= s["right"]) & (far >= -s["left"])
    window |= (far <= s["right"]) & (torch.arange(n, device="cuda") < s["sinks"])[None, :]
    place = far.clamp(-r, r) + r
    q, k, v = (s[x].double() for x in "qkv")
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    db = torch.zeros(h, 2 * r + 1, dtype=torch.float64, device="cuda")
    for i in range(b):
        seen = window if s["mask"] is None else window & s["mask"][i][None, :]
        some = seen.any(-1)
        for j in range(h):
            a = scale * (q[i, j] @ k[i, j // group].T)
            if r:
                a += s["rel_bias"][j].double()[place]
            a[~seen] = -math.inf
            p = torch.zeros_like(a)
            p[some] = torch.softmax(a[some], -1)
            o[i, j] = p @ v[i, j // group]
            if s["train"]:
                g = s["grad"][i, j].double()
                dv[i, j // group] += p.T @ g
                dp = g @ v[i, j // group].T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[i, j] = scale * (ds @ k[i, j // group])
                dk[i, j // group] += scale * (ds.T @ q[i, j])
                for c in range(-r, r + 1) if r else ():
                    db[j, c + r] += ds.diagonal(c).sum() if abs(c) < r else torch.triu(ds, r).sum() if c > 0 else torch.tril(ds, -r).sum()
    if not s["train"]:
        return o
    return (o, dq, dk, dv, db) if r else (o, dq, dk, dv)
