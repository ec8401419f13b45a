"""What the operators at the two ends of a training step cost: rotary positions of several axes in front of attention, a linear head with
softmax cross entropy that keeps no logits, and the orthogonalised update of weight matrices.

Heads of the pair representation classify every pair of tokens (64 distance bins over 128 channels), heads of the single one
a token (32 residue types over 384 channels) or an entry of a large vocabulary.  Rotary positions turn the queries and keys of local
attention (heads of 32 to 128, residue, atom and chain numbers as axes).  The update works on the weights of a stack at once: 48 blocks,
128 to 1536 rows and columns, or on single large matrices.

With ``own`` false, ``run`` is elementary tensor operations in 32 bits (angles and long sums in 64); with ``own`` true it makes the calls that a
user of the package makes.  Both take the same state.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)                 # of the update's odd polynomial of degree five
STEPS, EPS = 5, 1e-7


def listed():
    return [
        # Masked residues of one crop: few rows, few classes, most rows ignored; latency.
        {"name": "loss_residues_384", "op": "loss", "rows": 384, "c": 384, "v": 32, "bias": True, "smooth": 0.0, "ignored": 0.85,
         "dtype": "bf16", "train": True},
        # The distogram head of a complex of 768 tokens: every pair, 64 bins, padded pairs ignored.
        {"name": "loss_distogram_768", "op": "loss", "rows": 768 * 768, "c": 128, "v": 64, "bias": True, "smooth": 0.0, "ignored": 0.2,
         "dtype": "bf16", "train": True},
        # One short sequence scored against a large vocabulary, a loss for each token: forward alone, the weight is all there is to read.
        {"name": "loss_score_37", "op": "loss", "rows": 37, "c": 1024, "v": 65536, "bias": False, "smooth": 0.0, "ignored": 0.0,
         "dtype": "bf16", "train": False},
        # Odd numbers of rows and classes, smoothed labels, training in fp16.
        {"name": "loss_odd_train", "op": "loss", "rows": 3001, "c": 768, "v": 32003, "bias": True, "smooth": 0.1, "ignored": 0.1,
         "dtype": "fp16", "train": True},
        # A batch of long sequences over the largest vocabulary: training, bound by its products.
        {"name": "loss_large_train", "op": "loss", "rows": 8192, "c": 2048, "v": 131072, "bias": False, "smooth": 0.0, "ignored": 0.05,
         "dtype": "bf16", "train": True},
        # Queries and keys of one short chain in inference: latency.
        {"name": "rotary_short_97", "op": "rotary", "batch": 1, "n": 97, "heads": 4, "kv_heads": 4, "d": 32, "sections": "16", "far": 0,
         "interleaved": False, "per_axis": False, "dtype": "bf16", "train": False},
        # Atoms of five samples of a crop: residue, atom and chain as axes with a ladder of their own, fp32, odd length.
        {"name": "rotary_atoms_train", "op": "rotary", "batch": 5, "n": 3987, "heads": 4, "kv_heads": 4, "d": 32, "sections": "6,6,4", "far": 0,
         "interleaved": True, "per_axis": True, "dtype": "fp32", "train": True},
        # Three axes over one ladder, heads of k shared, positions far from zero: training.
        {"name": "rotary_axes_train", "op": "rotary", "batch": 2, "n": 16384, "heads": 16, "kv_heads": 4, "d": 128, "sections": "16,24,24",
         "far": 1000000, "interleaved": False, "per_axis": False, "dtype": "bf16", "train": True},
        # The square projections of a stack's pair path, one matrix a block, fp32 momentum.
        {"name": "update_pair_128", "op": "update", "batch": 48, "m": 128, "n": 128, "dtype": "fp32"},
        # The transitions of the pair path, four times as wide as high.
        {"name": "update_transition_512", "op": "update", "batch": 48, "m": 512, "n": 128, "dtype": "bf16"},
        # Transitions of the single representation.
        {"name": "update_single_1536", "op": "update", "batch": 24, "m": 384, "n": 1536, "dtype": "bf16"},
        # One large matrix.
        {"name": "update_large_4096", "op": "update", "batch": 1, "m": 4096, "n": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["loss", "loss", "rotary", "update"])
    if op == "loss":
        if rng.random() < 0.35:                           # heads over pairs or tokens with few classes
            rows, c, v = _log(rng, 1, 600000), rng.choice([64, 128]), _log(rng, 2, 128)
        else:
            c, v = 8 * _log(rng, 8, 256), _log(rng, 2, 131072)
            rows = max(1, min(_log(rng, 1, 32768), int(8192 * 2048 * 131072 / (c * v)), int(6e9 / (4 * v))))
        return {"op": op, "rows": rows, "c": c, "v": v, "bias": rng.random() < 0.5, "smooth": rng.choice([0.0, 0.0, 0.1]),
                "ignored": rng.choice([0.0, 0.15, 0.85]), "dtype": rng.choice(["bf16", "fp16"]), "train": rng.random() < 0.7}
    if op == "rotary":
        heads, kv_heads, d = rng.choice([(4, 4, 32), (16, 16, 24), (16, 16, 48), (8, 8, 64), (8, 2, 128), (16, 4, 64), (6, 2, 40), (8, 8, 256)])
        n = _log(rng, 1, 16384)
        batch = max(1, min(_log(rng, 1, 8), int(2 * 16384 * 20 * 128 / (n * (heads + kv_heads) * d))))
        pairs = rng.choice([d // 2, d // 2, d // 4])      # all of a head is turned, or its first half
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        return {"op": op, "batch": batch, "n": n, "heads": heads, "kv_heads": kv_heads, "d": d, "sections": ",".join(map(str, sections)),
                "far": rng.choice([0, 0, _log(rng, 1000, 10000000)]), "interleaved": rng.random() < 0.5, "per_axis": rng.random() < 0.5,
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "train": rng.random() < 0.6}
    m, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
    batch = max(1, min(_log(rng, 1, 64), int(4096 ** 3 / (min(m, n) ** 2 * max(m, n)))))
    # fp32 up to where products in 32 bits give a result that 32 bits are worth
    return {"op": op, "batch": batch, "m": m, "n": n, "dtype": rng.choice(["fp32", "bf16", "fp16"] if max(m, n) <= 1024 else ["bf16", "fp16"])}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "loss":
        rows, c, v = case["rows"], case["c"], case["v"]
        weight = _randn(g, v, c, dtype=dtype, std=2.0 / math.sqrt(c))
        target = torch.randint(0, v, (rows,), generator=g, device="cuda")
        # what a head sees half way through training: the row leans towards its class
        lean = 0.6 * c ** 0.5 / 2.0 * torch.rand(rows, 1, generator=g, device="cuda")
        x = (_randn(g, rows, c) + lean * weight[target].float()).to(dtype)
        ignored = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        s["target"] = target.masked_fill(ignored, IGNORE)
        s["target"][0] = 0                                # at least one row counts
        s["bias"] = _randn(g, v, dtype=dtype, std=0.5).requires_grad_(case["train"]) if case["bias"] else None
        s["x"], s["weight"] = x.requires_grad_(case["train"]), weight.requires_grad_(case["train"])
    elif case["op"] == "rotary":
        b, n, h, hk, d = (case[k] for k in ("batch", "n", "heads", "kv_heads", "d"))
        axes = len(case["sections"].split(","))
        # one projection gives q, k and v of all heads: the heads are views into its rows
        qkv = _randn(g, b, n, h + 2 * hk, d, dtype=dtype)
        q, k, _ = (t.transpose(1, 2) for t in qkv.split([h, hk, hk], dim=2))
        s["q"], s["k"] = (t.detach().requires_grad_(case["train"]) for t in (q, k))
        at = torch.arange(n, device="cuda")
        # running number, number within a group of about eight, number of a chain; samples begin at places of their own
        start = torch.randint(0, 50, (b, 1, axes), generator=g, device="cuda") + case["far"]
        s["positions"] = torch.stack([at, at % 8, at // 100][:axes], -1)[None] + start
        if case["train"]:
            s["grads"] = [_randn(g, b, n, x, d, dtype=dtype).transpose(1, 2) for x in (h, hk)]
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        # momentum: a few strong directions, a falling tail, and noise of the batches
        r = max(1, min(m, n) // 8)
        fall = torch.exp(-4.0 * torch.arange(r, device="cuda") / r)
        s["g"] = (((_randn(g, b, m, r) * fall) @ _randn(g, b, r, n) + 0.3 * _randn(g, b, m, n)) * 1e-3).to(dtype)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"loss": _plain_loss, "rotary": _plain_rotary, "update": _plain_update}[s["op"]](s)


def _sections(s):
    return tuple(int(x) for x in s["sections"].split(","))


def _own(s):
    import protenix_b200 as px

    if s["op"] == "loss":
        loss = px.linear_cross_entropy(s["x"], s["weight"], s["target"], bias=s["bias"], ignore_index=IGNORE, label_smoothing=s["smooth"],
                                       reduction="mean" if s["train"] else "none")
        if not s["train"]:
            return loss
        leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return loss.detach(), *torch.autograd.grad(loss, leaves)
    if s["op"] == "rotary":
        q, k = px.rotary_embedding(s["q"], s["k"], s["positions"], sections=_sections(s), interleaved=s["interleaved"], per_axis=s["per_axis"])
        if not s["train"]:
            return q, k
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), s["grads"])
    return px.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


def _plain_loss(s):
    x, w, eps, v = s["x"].float(), s["weight"].float(), s["smooth"], s["v"]
    logits = x @ w.t()
    if s["bias"] is not None:
        logits += s["bias"].float()
    counts = s["target"] != IGNORE
    at = s["target"].clamp_min(0)[:, None]
    top = logits.amax(-1, keepdim=True)
    hit, mean = logits.gather(1, at), logits.sum(-1, keepdim=True) / v if eps else 0.0
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    row = (total.log() + top - (1.0 - eps) * hit - eps * mean)[:, 0]
    row = torch.where(counts, row, 0.0)
    if not s["train"]:
        return row
    count = counts.sum()
    loss = (row.sum(dtype=torch.float64) / count).float()
    p /= total
    if eps:
        p -= eps / v
    p.scatter_add_(1, at, torch.full_like(hit, eps - 1.0))
    p *= (counts / count.float())[:, None]
    grads = [(p @ w).to(s["x"].dtype), (p.t() @ x).to(s["weight"].dtype)]
    if s["bias"] is not None:
        grads.append(p.sum(0, dtype=torch.float64).to(s["bias"].dtype))
    return loss, *grads


def _angles(s):
    """[B, 1, N, pairs] in 64 bits."""
    sections, out = _sections(s), []
    pairs, first = sum(sections), 0
    for axis, size in enumerate(sections):
        j = torch.arange(size, device="cuda", dtype=torch.float64)
        ladder = 10000.0 ** -(j / size if s["per_axis"] else (j + first) / pairs)
        out.append(s["positions"][..., axis, None].double() * ladder)
        first += size
    return torch.cat(out, -1)[:, None]


def _turn(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    y = x.float().clone()
    a = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    b = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    u, v = x[..., a].float(), x[..., b].float()
    y[..., a] = u * cos - v * sin
    y[..., b] = v * cos + u * sin
    return y.to(x.dtype)


def _plain_rotary(s):
    angle = _angles(s)
    cos, sin = angle.cos().float(), angle.sin().float()
    out = [_turn(s[x], cos, sin, s["interleaved"]) for x in "qk"]
    if s["train"]:
        out += [_turn(g, cos, -sin, s["interleaved"]) for g in s["grads"]]
    return tuple(out)


def _plain_update(s):
    x = s["g"].float()
    wide = s["m"] <= s["n"]
    if not wide:
        x = x.transpose(-1, -2)
    a, b, c = COEFFICIENTS
    x = x / (x.square().sum((-2, -1), keepdim=True, dtype=torch.float64).sqrt().float() + EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x if wide else x.transpose(-1, -2)).to(s["g"].dtype).contiguous()


# ---- work and exact values -------------------------------------------------------------------------------------------
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "loss":
        r, c, v = case["rows"], case["c"], case["v"]
        operands = (r * c + v * c + (v if case["bias"] else 0)) * size
        passes = 2 if case["train"] else 1                # gradients are as large as what they belong to
        return {"bytes": passes * operands + 8 * r, "flops": (6 if case["train"] else 2) * r * v * c}
    if case["op"] == "rotary":
        rows = case["batch"] * case["n"]
        elements, pairs = rows * (case["heads"] + case["kv_heads"]) * case["d"], sum(_sections(case))
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * elements * size + 8 * rows * case["sections"].count(",") + 8 * rows,
                "flops": passes * 6 * rows * (case["heads"] + case["kv_heads"]) * pairs}
    m, n = sorted((case["m"], case["n"]))
    # the two symmetric products need half of their elements
    step = m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n
    return {"bytes": 2 * case["batch"] * m * n * size, "flops": case["batch"] * STEPS * step}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"loss": _exact_loss, "rotary": _exact_rotary, "update": _exact_update}[s["op"]](s)


def _exact_loss(s):
    """A block of rows at a time; the gradient as the smoothed one-hot vector's distance from the softmax."""
    w, eps, v = s["weight"].double(), s["smooth"], s["v"]
    keep = torch.nonzero(s["target"] != IGNORE)[:, 0]
    each = torch.zeros(s["rows"], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.zeros_like(s["x"], dtype=torch.float64), torch.zeros_like(w), torch.zeros(v, dtype=torch.float64, device="cuda")
    for at in keep.split(max(256, 2 ** 27 // v)):
        x, t = s["x"][at].double(), s["target"][at]
        logits = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
        log_p = torch.log_softmax(logits, -1)
        want = torch.full_like(log_p, eps / v)
        want[torch.arange(len(at), device="cuda"), t] += 1.0 - eps
        each[at] = -(want * log_p).sum(-1)
        if s["train"]:
            dl = (log_p.exp() - want) / len(keep)
            dx[at] = dl @ w
            dw += dl.t() @ x
            db += dl.sum(0)
    if not s["train"]:
        return each
    loss = each.sum() / len(keep)
    return (loss, dx, dw) if s["bias"] is None else (loss, dx, dw, db)


def _exact_rotary(s):
    """Pairs as complex numbers, multiplied by a number on the unit circle."""
    sections = _sections(s)
    p = sum(sections)
    step = [(j / n if s["per_axis"] else (j + sum(sections[:a])) / p, a) for a, n in enumerate(sections) for j in range(n)]
    speed = torch.tensor([math.exp(-math.log(10000.0) * x) for x, _ in step], dtype=torch.float64, device="cuda")
    angle = s["positions"].double()[..., [a for _, a in step]] * speed
    circle = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x, by):
        y = x.double()
        pairs = y[..., : 2 * p]
        pairs = pairs.unflatten(-1, (p, 2)) if s["interleaved"] else torch.stack(pairs.split(p, -1), -1)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z.flatten(-2) if s["interleaved"] else torch.cat([z[..., 0], z[..., 1]], -1)
        return torch.cat([z, y[..., 2 * p:]], -1)

    out = [turned(s[x], circle) for x in "qk"]
    return tuple(out + [turned(g, circle.conj()) for g in s["grads"]] if s["train"] else out)


def _exact_update(s):
    """The polynomial by Horner's rule on the smaller Gram matrix, from the side that this leaves."""
    x = s["g"].double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS)
    a, b, c = COEFFICIENTS
    one = torch.eye(min(s["m"], s["n"]), dtype=torch.float64, device="cuda")
    for _ in range(STEPS):
        if s["m"] < s["n"]:
            gram = torch.matmul(x, x.mT)
            x = torch.matmul(torch.matmul(b * one + c * gram, gram) + a * one, x)
        else:
            gram = torch.matmul(x.mT, x)
            x = torch.matmul(x, torch.matmul(b * one + c * gram, gram) + a * one)
    return x
