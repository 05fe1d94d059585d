"""Timing cases of three operators of the training step.

``group_norm``  normalisation over channel groups of a channels-last activation, with the residual
                add and the activation in the same pass, and its gradients
                (``ops.functional.group_norm_act``)
``linear_xent`` mean softmax cross-entropy of a classifier over many classes, straight from the
                features and the classifier's weight, with its gradients and the top-1 count
                (``ops.functional.linear_cross_entropy``)
``ns``          Newton-Schulz orthogonalisation of weight updates, one matrix or the matrices of a
                whole model in one call (``ops.functional.newton_schulz``)

``run`` computes a case in its plain form (elementary torch operations in fp32) or, with ``own``,
through the framework's entry points.  ``exact`` computes the same outputs in fp64 from the
definitions.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
IGNORE = -100


# ---------------------------------------------------------------------------- cases
def _gn(name, n, h, w, c, g, dtype, act, res, train):
    return {"name": name, "op": "group_norm", "n": n, "h": h, "w": w, "c": c, "groups": g,
            "dtype": dtype, "act": act, "residual": res, "train": train}


def _ce(name, n, d, v, dtype, ignored, train):
    return {"name": name, "op": "linear_xent", "n": n, "d": d, "v": v, "dtype": dtype,
            "ignored": ignored, "train": train}


def _ns(name, shapes, dtype):
    return {"name": name, "op": "ns", "shapes": shapes, "dtype": dtype}


# the convolution weights of ResNet-50 as [out channels, kernel * kernel * in channels] matrices
def _resnet50_matrices():
    out, cin = [(64, 49 * 3)], 64
    for planes, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for b in range(blocks):
            out += [(planes, cin), (planes, 9 * planes), (4 * planes, planes)]
            if b == 0:
                out.append((4 * planes, cin))
            cin = 4 * planes
    return out


def _text(shapes):
    return ",".join(f"{m}x{n}" for m, n in shapes)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def listed():
    return [
        # one image through the last CIFAR stage at evaluation: a call's latency
        _gn("gn_eval_one_image", 1, 4, 4, 512, 32, "bf16", "relu", False, False),
        # ResNet-50's first-stage block output at batch 256: residual add and ReLU in the same pass
        _gn("gn_block_56", 256, 56, 56, 256, 32, "bf16", "relu", True, True),
        # the stem's 112 x 112 activation at batch 64, two channels to a group
        _gn("gn_stem_112", 64, 112, 112, 64, 32, "bf16", "relu", False, True),
        # fp32 activations of an odd size, groups of 12 channels, the smooth activation
        _gn("gn_fp32_odd", 7, 33, 29, 120, 10, "fp32", "silu", False, True),
        # the CIFAR classifier at the per-GPU batch of 32: a call's latency
        _ce("xent_cifar", 32, 512, 10, "bf16", 0, True),
        # the ImageNet classifier of ResNet-50 at batch 256
        _ce("xent_imagenet", 256, 2048, 1000, "bf16", 0, True),
        # fp32 operands, odd sizes, some rows without a label
        _ce("xent_fp32_odd", 197, 300, 10007, "fp32", 23, True),
        # a vocabulary of 131,072 classes, 8,192 rows, a few of them padding
        _ce("xent_vocab_128k", 8192, 2048, 131072, "bf16", 100, True),
        # the stem's 64 x 27 weight of the CIFAR network alone: a call's latency
        _ns("ns_cifar_stem", _text([(64, 27)]), "fp32"),
        # the largest 3 x 3 weight of ResNet-50 alone
        _ns("ns_conv_512", _text([(512, 4608)]), "fp32"),
        # every convolution weight of ResNet-50, as one optimizer step hands them over
        _ns("ns_resnet50", _text(_resnet50_matrices()), "fp32"),
        # one large square matrix in bf16
        _ns("ns_4096", _text([(4096, 4096)]), "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm", "linear_xent", "ns"])
    dtype = rng.choice(["bf16", "fp32"])
    if op == "group_norm":
        while True:
            g, cg = rng.choice([1, 2, 5, 8, 16, 32]), _log_int(rng, 1, 64)
            n, h, w = _log_int(rng, 1, 256), _log_int(rng, 1, 112), _log_int(rng, 1, 112)
            if n * h * w * g * cg <= (256 * 56 * 56 * 256) // (1 if dtype == "bf16" else 2):
                return {k: v for k, v in _gn("", n, h, w, g * cg, g, dtype,
                                             rng.choice(["none", "relu", "silu"]), rng.random() < 0.5,
                                             rng.random() < 0.75).items() if k != "name"}
    if op == "linear_xent":
        while True:
            n, d, v = _log_int(rng, 1, 8192), _log_int(rng, 8, 4096), _log_int(rng, 2, 131072)
            if n * d * v <= (8192 * 2048 * 131072) // (1 if dtype == "bf16" else 8):
                return {k: v_ for k, v_ in _ce("", n, d, v, dtype, rng.randrange(0, n // 4 + 1),
                                               rng.random() < 0.75).items() if k != "name"}
    while True:
        shapes = [(_log_int(rng, 1, 4096), _log_int(rng, 1, 4096)) for _ in range(rng.choice([1, 1, 2, 5, 9]))]
        if sum(min(m, n) ** 2 * max(m, n) for m, n in shapes) <= 4096 ** 3:
            return {k: v for k, v in _ns("", _text(shapes), dtype).items() if k != "name"}


# --------------------------------------------------------------------------- inputs
def _randn(shape, gen, scale=1.0, dtype=torch.float32):
    # made in slices: the fp32 draw of a large activation is never whole in memory
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        part = flat[i:i + (1 << 26)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEV) * scale)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"case": dict(case)}
    if case["op"] == "group_norm":
        dt = _DT[case["dtype"]]
        shape = (case["n"], case["h"], case["w"], case["c"])
        # convolution outputs: every channel with a mean and a width of its own
        mean = torch.randn(case["c"], generator=gen, device=DEV)
        width = torch.rand(case["c"], generator=gen, device=DEV) + 0.5
        x = _randn(shape, gen, dtype=dt)
        for i in range(0, shape[0], 32):
            x[i:i + 32] = (x[i:i + 32].float() * width + mean).to(dt)
        gn = torch.nn.GroupNorm(case["groups"], case["c"], eps=1e-5, device=DEV)
        with torch.no_grad():
            gn.weight.copy_(torch.rand(case["c"], generator=gen, device=DEV) + 0.5)
            gn.bias.copy_(torch.randn(case["c"], generator=gen, device=DEV) * 0.2)
        st["gn"], st["x"] = gn, x
        st["res"] = _randn(shape, gen, dtype=dt) if case["residual"] else None
        if case["train"]:
            # gradients as they come down from the pooled classifier: a mean to every channel
            lean = torch.randn(case["c"], generator=gen, device=DEV) * 1e-2
            dy = _randn(shape, gen, 1e-2, dt)
            for i in range(0, shape[0], 32):
                dy[i:i + 32] = (dy[i:i + 32].float() + lean).to(dt)
            st["dy"] = dy
            x.requires_grad_(True)
            if case["residual"]:
                st["res"].requires_grad_(True)
    elif case["op"] == "linear_xent":
        dt = _DT[case["dtype"]]
        n, d, v = case["n"], case["d"], case["v"]
        lin = torch.nn.Linear(d, v, device="meta").to_empty(device=DEV).to(dt)
        with torch.no_grad():
            lin.weight.copy_(_randn((v, d), gen, 1.0 / math.sqrt(d), dt))
            lin.bias.copy_(torch.randn(v, generator=gen, device=DEV) * 0.1)
        target = torch.randint(0, v, (n,), generator=gen, device=DEV)
        # half of the rows know their class (a clear margin), the other half do not yet
        x = torch.randn(n, d, generator=gen, device=DEV)
        known = (torch.arange(n, device=DEV) % 2 == 0).float()[:, None]
        x = x + known * 12.0 * lin.weight.detach()[target].float()
        if case["ignored"]:
            rows = torch.randperm(n, generator=gen, device=DEV)[:case["ignored"]]
            target[rows] = IGNORE
        x = x.to(dt)
        if case["train"]:
            x.requires_grad_(True)
            st["gloss"] = torch.ones((), device=DEV)
        st.update(lin=lin, x=x, target=target)
    else:
        mats = []
        for m, n in _shapes(case):
            # an averaged gradient: a few strong directions over a broad floor
            r = max(1, min(m, n) // 16)
            a = torch.randn(m, r, generator=gen, device=DEV)
            b = torch.randn(r, n, generator=gen, device=DEV)
            u = (a @ b) * (0.3 / math.sqrt(r)) + torch.randn(m, n, generator=gen, device=DEV)
            mats.append((u * 1e-3).to(_DT[case["dtype"]]))
        st["mats"] = mats
    return st


# ---------------------------------------------------------------------- plain forms
def _plain_gn(st):
    c = st["case"]
    x, gn, res = st["x"].detach(), st["gn"], st["res"]
    n, g, ch = c["n"], c["groups"], c["c"]
    cg = ch // g
    xf = x.float().reshape(n, -1, g, cg)
    mean = xf.mean(dim=(1, 3), keepdim=True)
    xc = xf - mean
    rstd = torch.rsqrt((xc * xc).mean(dim=(1, 3), keepdim=True) + gn.eps)
    xhat = xc * rstd
    del xf, xc
    gamma, beta = gn.weight.detach().reshape(g, cg), gn.bias.detach().reshape(g, cg)
    z = xhat * gamma + beta
    if res is not None:
        z = z + res.detach().float().reshape(n, -1, g, cg)
    if c["act"] == "relu":
        out = z.clamp_min(0.0)
    elif c["act"] == "silu":
        out = z * torch.sigmoid(z)
    else:
        out = z
    out = out.to(x.dtype).reshape(x.shape)
    if not c["train"]:
        return out
    dz = st["dy"].float().reshape(n, -1, g, cg)
    if c["act"] == "relu":
        dz = dz * (z > 0)
    elif c["act"] == "silu":
        s = torch.sigmoid(z)
        dz = dz * (s * (1.0 + z * (1.0 - s)))
    del z
    dres = dz.to(x.dtype).reshape(x.shape) if res is not None else None
    # sums over every pixel of the batch, whose terms cancel: in fp64
    dgamma = (dz * xhat).sum(dim=(0, 1), dtype=torch.float64).float().reshape(ch)
    dbeta = dz.sum(dim=(0, 1), dtype=torch.float64).float().reshape(ch)
    dh = dz * gamma
    del dz
    m1 = dh.mean(dim=(1, 3), keepdim=True)
    m2 = (dh * xhat).mean(dim=(1, 3), keepdim=True)
    dx = ((dh - m1 - xhat * m2) * rstd).to(x.dtype).reshape(x.shape)
    outs = [out, dx, dgamma, dbeta]
    return outs + [dres] if res is not None else outs


def _plain_xent(st):
    c = st["case"]
    x, lin, target = st["x"].detach(), st["lin"], st["target"]
    w, b = lin.weight.detach().float(), lin.bias.detach().float()
    logits = x.float() @ w.t() + b
    keep = target != IGNORE
    count = keep.sum().clamp_min(1)
    t = torch.where(keep, target, torch.zeros_like(target))
    top = logits.max(dim=1, keepdim=True)
    correct = ((top.indices[:, 0] == t) & keep).sum().reshape(1)
    e = torch.exp(logits - top.values)
    s = e.sum(dim=1, keepdim=True)
    lt = logits.gather(1, t[:, None])
    loss = torch.where(keep, (torch.log(s) + top.values - lt)[:, 0], torch.zeros((), device=x.device)).sum() / count
    del logits
    if not c["train"]:
        return [loss, correct]
    p = e.div_(s)
    p.scatter_add_(1, t[:, None], torch.full_like(lt, -1.0))
    p.mul_(keep.float()[:, None] * (st["gloss"] / count))
    dx = (p @ w).to(x.dtype)
    dw = (p.t() @ x.float()).to(lin.weight.dtype)
    db = p.sum(dim=0, dtype=torch.float64).to(lin.bias.dtype)
    return [loss, correct, dx, dw, db]


def _plain_ns(st):
    a, b, c = NS_COEFFS
    out = []
    for u in st["mats"]:
        x = u.float()
        tall = x.shape[0] > x.shape[1]
        if tall:
            x = x.t()
        x = x / (torch.sqrt((x * x).sum()) + NS_EPS)
        for _ in range(NS_STEPS):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        out.append((x.t() if tall else x).contiguous().to(u.dtype))
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"group_norm": _plain_gn, "linear_xent": _plain_xent, "ns": _plain_ns}[c["op"]](state)
    from pytorch_multiprocessing_distributed_amd.ops import functional as OF
    if c["op"] == "group_norm":
        x, gn, res = state["x"], state["gn"], state["res"]
        if not c["train"]:
            with torch.no_grad():
                return OF.group_norm_act(x, gn, residual=res, act=c["act"])
        out = OF.group_norm_act(x, gn, residual=res, act=c["act"])
        leaves = [x, gn.weight, gn.bias] + ([res] if res is not None else [])
        return [out.detach(), *torch.autograd.grad(out, leaves, state["dy"])]
    if c["op"] == "linear_xent":
        x, lin = state["x"], state["lin"]
        if not c["train"]:
            with torch.no_grad():
                loss, correct = OF.linear_cross_entropy(x, lin, state["target"], ignore_index=IGNORE)
            return [loss, correct]
        loss, correct = OF.linear_cross_entropy(x, lin, state["target"], ignore_index=IGNORE)
        grads = torch.autograd.grad(loss, [x, lin.weight, lin.bias], state["gloss"])
        return [loss.detach(), correct, *grads]
    return OF.newton_schulz(state["mats"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)


# ---------------------------------------------------------------------------- exact
def _exact_gn(c, st):
    x = st["x"].detach().double()
    n, ch, g = c["n"], c["c"], c["groups"]
    rows = x.reshape(n, -1, ch)
    per = rows.shape[1] * (ch // g)

    def over_group(t):                      # [n, pixels, ch] -> the group's sum at every channel
        s = t.sum(1).reshape(n, g, ch // g).sum(2)
        return s.repeat_interleave(ch // g, dim=1)[:, None, :]

    mu = over_group(rows) / per
    var = over_group((rows - mu).square()) / per
    inv = 1.0 / torch.sqrt(var + st["gn"].eps)
    h = (rows - mu).mul_(inv)
    w, b = st["gn"].weight.detach().double(), st["gn"].bias.detach().double()
    z = h * w + b
    if st["res"] is not None:
        z += st["res"].detach().double().reshape(z.shape)
    sig = 1.0 / (1.0 + torch.exp(-z)) if c["act"] == "silu" else None
    act = {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * sig}[c["act"]]()
    out = act.reshape(x.shape)
    if not c["train"]:
        return out
    slope = {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(),
             "silu": lambda: sig + z * sig * (1.0 - sig)}[c["act"]]()
    dz = slope.mul_(st["dy"].double().reshape(z.shape))
    dh = dz * w
    dx = inv * (dh - over_group(dh) / per - h * (over_group(dh * h) / per))
    outs = [out, dx.reshape(x.shape), (dz * h).sum((0, 1)), dz.sum((0, 1))]
    if st["res"] is not None:
        outs.append(dz.reshape(x.shape))
    return outs


def _exact_xent(c, st):
    x, w = st["x"].detach().double(), st["lin"].weight.detach().double()
    bias, target = st["lin"].bias.detach().double(), st["target"]
    rows = torch.nonzero(target != IGNORE)[:, 0]
    cnt = max(1, rows.numel())
    loss = torch.zeros((), dtype=torch.float64, device=x.device)
    correct = torch.zeros(1, dtype=torch.int64, device=x.device)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for part in rows.split(2048):
        xi, ti = x[part], target[part]
        logit = torch.addmm(bias, xi, w.t())
        lse = torch.logsumexp(logit, dim=1)
        pick = torch.arange(part.numel(), device=x.device)
        loss += (lse - logit[pick, ti]).sum() / cnt
        correct += (logit.argmax(1) == ti).sum()
        if c["train"]:
            q = torch.exp(logit - lse[:, None])
            q[pick, ti] -= 1.0
            q /= cnt
            dx[part] = q @ w
            dw += q.t() @ xi
            db += q.sum(0)
    return [loss, correct, dx, dw, db] if c["train"] else [loss, correct]


def _exact_ns(c, st):
    outs = []
    for u in st["mats"]:
        y = u.double()
        flip = y.shape[0] > y.shape[1]
        y = y.mT if flip else y
        y = y / (torch.linalg.matrix_norm(y) + NS_EPS)
        for _ in range(NS_STEPS):
            gram = y @ y.mT
            poly = NS_COEFFS[1] * gram + NS_COEFFS[2] * (gram @ gram)
            y = NS_COEFFS[0] * y + poly @ y
        outs.append(y.mT.contiguous() if flip else y)
    return outs


def exact(case, seed):
    st = prepare(case, seed)
    return {"group_norm": _exact_gn, "linear_xent": _exact_xent, "ns": _exact_ns}[case["op"]](case, st)


# ----------------------------------------------------------------------------- work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "group_norm":
        el = case["n"] * case["h"] * case["w"] * case["c"]
        tensors = 2 + (1 if case["residual"] else 0)              # x, out, residual
        flops = 8 * el
        if case["train"]:
            tensors += 2 + (1 if case["residual"] else 0)         # dy, dx, dresidual
            flops += 14 * el
        return {"bytes": tensors * el * e + 16 * case["c"], "flops": flops}
    if case["op"] == "linear_xent":
        n, d, v = case["n"], case["d"], case["v"]
        operands = (n * d + v * d + v) * e
        if case["train"]:
            return {"bytes": 2 * operands + 8 * n, "flops": 6 * n * d * v}
        return {"bytes": operands + 8 * n, "flops": 2 * n * d * v}
    nbytes = flops = 0
    for m, n in _shapes(case):
        s, l = min(m, n), max(m, n)
        nbytes += 2 * m * n * e
        # the two symmetric products need one triangle each
        flops += NS_STEPS * (s * (s + 1) * l + s * s * (s + 1) + 2 * s * s * l)
    return {"bytes": nbytes, "flops": flops}
