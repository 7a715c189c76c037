"""Calls that time the normalisation, attention and dropout operators of a segmentation decoder.

Three operators, each with its backward pass:

* ``group_norm_act``   group normalisation of a channels-last map, then a residual, then an activation
* ``cross_attention``  queries of one length over the keys and values of another (a decoder's positions over an encoder's)
* ``dropout``          dropout whose mask is a function of (seed, position) and is never stored

``run`` computes them either in plain torch operations (``own`` false) or through the framework's entry points
(``own`` true); ``exact`` is the same from the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one 513 x 513 image at stride 16, after the pyramid's projection: prediction, where the launch counts
        {"name": "norm one image", "op": "norm", "type": "bf16", "n": 1, "c": 256, "h": 33, "w": 33, "groups": 32,
         "act": "relu", "residual": False, "train": False},
        # the projection of the low-level features has 48 channels: three to a group; fp32 training, block with identity
        {"name": "norm fp32 48 channels", "op": "norm", "type": "fp32", "n": 3, "c": 48, "h": 65, "w": 97, "groups": 16,
         "act": "relu", "residual": True, "train": True},
        # a dual-attention head on 512 x 512 images at stride 8, 16 images to a step
        {"name": "norm attention head", "op": "norm", "type": "bf16", "n": 16, "c": 512, "h": 64, "w": 64, "groups": 32,
         "act": "relu", "residual": False, "train": True},
        # the decoder at stride 4 of 513 x 513 images, 16 to a step: far larger than the last-level cache
        {"name": "norm decoder", "op": "norm", "type": "bf16", "n": 16, "c": 256, "h": 129, "w": 129, "groups": 32,
         "act": "silu", "residual": False, "train": True},
        # one query an image over an encoder's map (interactive prediction): shared heads, ragged maps
        {"name": "attention one query", "op": "attention", "type": "bf16", "b": 8, "lq": 1, "lk": 4225, "heads": 8,
         "kv_heads": 2, "dim": 128, "lengths": "4225,4225,1089,2048,3000,4224,17,4097", "masked": 0.0, "train": False},
        # ragged encoder maps, one of them empty, a mask inside the others; shared heads, fp16, odd lengths and width
        {"name": "attention ragged", "op": "attention", "type": "fp16", "b": 5, "lq": 1089, "lk": 777, "heads": 8,
         "kv_heads": 2, "dim": 96, "lengths": "777,0,401,1,640", "masked": 0.2, "train": True},
        # a training step's decoder: stride-4 positions over the stride-16 map of 513 x 513 images
        {"name": "attention decoder", "op": "attention", "type": "bf16", "b": 16, "lq": 16641, "lk": 1089, "heads": 4,
         "kv_heads": 4, "dim": 64, "lengths": "", "masked": 0.0, "train": True},
        # prediction on a large image: every stride-8 position over a stride-4 map
        {"name": "attention long", "op": "attention", "type": "bf16", "b": 1, "lq": 4225, "lk": 16641, "heads": 8,
         "kv_heads": 8, "dim": 128, "lengths": "", "masked": 0.0, "train": False},
        # the classifier's input of one image
        {"name": "dropout one image", "op": "dropout", "type": "bf16", "n": 1, "c": 256, "h": 33, "w": 33, "p": 0.1,
         "residual": False, "device_seed": False, "train": True},
        # fp32 logits of 21 classes: an odd number of elements; the seed lives on the device, as a captured step holds it
        {"name": "dropout fp32 21 classes", "op": "dropout", "type": "fp32", "n": 7, "c": 21, "h": 129, "w": 129,
         "p": 0.25, "residual": False, "device_seed": True, "train": True},
        # the decoder's map at stride 4, 16 images to a step, added to the identity branch
        {"name": "dropout decoder", "op": "dropout", "type": "bf16", "n": 16, "c": 256, "h": 129, "w": 129, "p": 0.5,
         "residual": True, "device_seed": False, "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "attention", "dropout"))
    if op == "attention":
        dim = rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * rng.choice((1, 1, 2, 4))
        train = rng.random() < 0.6
        b = _log_int(rng, 1, 16)
        lq = 1 if rng.random() < 0.2 else _log_int(rng, 2, 16641)
        lk = _log_int(rng, 1, 16641)
        pairs = 16.0 * 4 * 16641 * 1089                         # of the largest listed step, in products and in scores
        while b * heads * lq * lk > pairs or (14.0 if train else 4.0) * b * heads * lq * lk * dim > 14.0 * pairs * 64:
            lq, lk, b = max(1, lq * 2 // 3), max(1, lk * 2 // 3), max(1, b * 3 // 4)
        lengths = ""
        if rng.random() < 0.6:
            lengths = ",".join(str(lk if rng.random() < 0.3 else rng.randint(0, lk)) for _ in range(b))
        return {"op": op, "type": rng.choice(("bf16", "fp16")), "b": b, "lq": lq, "lk": lk, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "lengths": lengths, "masked": rng.choice((0.0, 0.0, 0.1, 0.5)),
                "train": train}
    c = rng.choice((1, 3, 21, 48, 64, 96, 128, 256, 304, 320, 512, 728, 1024, 2048))
    n, h, w = _log_int(rng, 1, 32), _log_int(rng, 1, 129), _log_int(rng, 1, 129)
    kind = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    largest = 16 * 256 * 129 * 129 // (2 if kind == "fp32" else 1)
    while n * c * h * w > largest:
        n, h, w = max(1, n * 2 // 3), max(1, h * 3 // 4), max(1, w * 3 // 4)
    case = {"op": op, "type": kind, "n": n, "c": c, "h": h, "w": w, "residual": rng.random() < 0.4}
    if op == "norm":
        whole = [g for g in (1, 2, 3, 4, 7, 8, 16, 32, 64, c) if c % g == 0]
        case.update(groups=rng.choice(whole), act=rng.choice(("none", "relu", "silu")), train=rng.random() < 0.7)
    else:
        case.update(p=rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)), device_seed=rng.random() < 0.5, train=True)
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _map(gen, case, kind, spread=1.0):
    t = torch.randn((case["n"], case["h"], case["w"], case["c"]), generator=gen, device="cuda") * spread
    return t.to(kind).permute(0, 3, 1, 2)                      # [n, c, h, w], channels last


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "attention":
        b, lq, lk, hq, hk, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
        shape = {"q": (b, lq, hq, d), "k": (b, lk, hk, d), "v": (b, lk, hk, d)}
        if case["train"]:
            shape["dout"] = (b, lq, hq, d)
        for name, sh in shape.items():
            s[name] = torch.randn(sh, generator=gen, device="cuda").to(kind)
        s["lengths"] = None
        if case["lengths"]:
            s["lengths"] = torch.tensor([int(t) for t in case["lengths"].split(",")], dtype=torch.int32, device="cuda")
        s["mask"] = None
        if case["masked"]:
            s["mask"] = torch.rand((b, lk), generator=gen, device="cuda") >= case["masked"]
        leaves = ("q", "k", "v")
    elif case["op"] == "norm":
        c = case["c"]
        # what a convolution leaves: every channel with a mean and a spread of its own
        shift = torch.randn((1, c, 1, 1), generator=gen, device="cuda")
        spread = 0.5 + torch.rand((1, c, 1, 1), generator=gen, device="cuda")
        x = _map(gen, case, torch.float32) * spread + shift
        s["x"] = x.to(kind)
        s["weight"] = 1.0 + 0.2 * torch.randn(c, generator=gen, device="cuda")
        s["bias"] = 0.2 * torch.randn(c, generator=gen, device="cuda")
        s["residual"] = _map(gen, case, kind) if case["residual"] else None
        if case["train"]:
            s["dout"] = _map(gen, case, kind)
        leaves = ("x", "weight", "bias", "residual")
    else:
        s["x"] = _map(gen, case, kind)
        s["residual"] = _map(gen, case, kind) if case["residual"] else None
        s["dout"] = _map(gen, case, kind)
        number = torch.randint(0, 1 << 62, (1,), generator=gen, device="cuda", dtype=torch.int64)
        s["seed"] = number if case["device_seed"] else int(number.item())
        leaves = ("x", "residual")
    s["leaves"] = [s[k] for k in leaves if s[k] is not None]
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(case, state)
        if case["op"] == "attention":
            return _plain_attention(case, state)
        return _plain_dropout(case, state)


def _run_own(case, s):
    from distributedpytorch_amd import ops
    if case["op"] == "norm":
        out = ops.group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], _EPS, act=case["act"],
                                 residual=s["residual"])
    elif case["op"] == "attention":
        out = ops.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["lengths"], key_mask=s["mask"])
    else:
        out = ops.dropout(s["x"], case["p"], seed=s["seed"], residual=s["residual"])
    if not case["train"]:
        return (out,)
    return (out.detach(),) + torch.autograd.grad(out, s["leaves"], s["dout"])


def _plain_norm(case, s):
    n, c, h, w = s["x"].shape
    g = case["groups"]
    kind = s["x"].dtype

    def split(t):                                               # [n, g, c/g, h*w]
        return t.float().reshape(n, g, c // g, h * w)

    x = split(s["x"])
    mean = x.mean(dim=(2, 3), keepdim=True)
    var = ((x - mean) ** 2).mean(dim=(2, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + _EPS)
    xhat = (x - mean) * rstd
    weight, bias = s["weight"].reshape(1, g, c // g, 1), s["bias"].reshape(1, g, c // g, 1)
    z = xhat * weight + bias
    if s["residual"] is not None:
        z = z + split(s["residual"])
    if case["act"] == "relu":
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif case["act"] == "silu":
        y = z / (1.0 + torch.exp(-z))
    else:
        y = z
    y = y.reshape(n, c, h, w).to(kind)
    if not case["train"]:
        return (y,)
    dz = split(s["dout"])
    if case["act"] == "relu":
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif case["act"] == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * sig * (1.0 + z * (1.0 - sig))
    dweight = (dz * xhat).sum(dim=(0, 3)).reshape(c)
    dbias = dz.sum(dim=(0, 3)).reshape(c)
    dxhat = dz * weight
    m1 = dxhat.mean(dim=(2, 3), keepdim=True)
    m2 = (dxhat * xhat).mean(dim=(2, 3), keepdim=True)
    dx = rstd * (dxhat - m1 - xhat * m2)
    out = (y, dx.reshape(n, c, h, w).to(kind), dweight, dbias)
    return out + ((dz.reshape(n, c, h, w).to(kind),) if s["residual"] is not None else ())


def _plain_attention(case, s):
    kind = s["q"].dtype
    hq, hk, d, lk = case["heads"], case["kv_heads"], case["dim"], case["lk"]
    share = hq // hk
    scale = 1.0 / math.sqrt(d)
    allowed = torch.ones((case["b"], lk), dtype=torch.bool, device=s["q"].device)
    if s["lengths"] is not None:
        allowed = allowed & (torch.arange(lk, device=s["q"].device) < s["lengths"][:, None])
    if s["mask"] is not None:
        allowed = allowed & s["mask"]

    def heads_first(t, kv):                                     # [b, l, h, d] -> [b, hq, l, d]
        t = t.float()
        if kv:
            t = torch.where(allowed[:, :, None, None], t, torch.zeros_like(t)).repeat_interleave(share, dim=2)
        return t.permute(0, 2, 1, 3).contiguous()

    q, k, v = heads_first(s["q"], False), heads_first(s["k"], True), heads_first(s["v"], True)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    score.masked_fill_(~allowed[:, None, None, :], float("-inf"))
    top = score.max(dim=3, keepdim=True)[0]
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    prob = torch.exp(score - top)
    total = prob.sum(dim=3, keepdim=True)
    prob /= torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(prob, v)

    def back(t, kv):                                            # [b, hq, l, d] -> [b, l, h, d]
        t = t.permute(0, 2, 1, 3)
        if kv:
            t = t.reshape(t.shape[0], t.shape[1], hk, share, d).sum(dim=3)
        return t.contiguous().to(kind)

    if not case["train"]:
        return (back(out, False),)
    do = heads_first(s["dout"], False)
    dv = torch.matmul(prob.transpose(2, 3).contiguous(), do)
    dprob = torch.matmul(do, v.transpose(2, 3).contiguous())
    dscore = prob * (dprob - (do * out).sum(dim=3, keepdim=True)) * scale
    dq = torch.matmul(dscore, k)
    dk = torch.matmul(dscore.transpose(2, 3).contiguous(), q)
    return back(out, False), back(dq, False), back(dk, True), back(dv, True)


_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _threshold(p):
    return min(65535, max(1, int(round(p * 65536))))


def _plain_keep(count, seed, p, device):
    """Philox4x32, ten rounds: block i of eight elements has the counter (i, i >> 32, 0, 0) and the seed as its key;
    each of the four words decides two elements, its low half the first.  An element stays where its half reaches
    the threshold."""
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    a, b = block & _LOW, block >> 32
    c, d = torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        left, right = a * _M0, c * _M1
        a, b, c, d = (((right >> 32) & _LOW) ^ b ^ k0), right & _LOW, (((left >> 32) & _LOW) ^ d ^ k1), left & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    words = torch.stack((a, b, c, d), dim=1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=2)
    return halves.reshape(-1)[:count] >= _threshold(p)


def _plain_dropout(case, s):
    x = s["x"]
    kind = x.dtype
    n, c, h, w = x.shape
    keep = _plain_keep(x.numel(), s["seed"], case["p"], x.device).reshape(n, h, w, c).permute(0, 3, 1, 2)
    factor = 65536.0 / (65536.0 - _threshold(case["p"]))
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * factor, zero)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    dx = torch.where(keep, s["dout"].float() * factor, zero).to(kind)
    return (y.to(kind), dx) + ((s["dout"],) if s["residual"] is not None else ())


# ---------------------------------------------------------------------------------------------------- what it has to do
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "attention":
        b, lq, lk, hq, hk, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
        keys = sum(int(t) for t in case["lengths"].split(",")) if case["lengths"] else b * lk
        seen = keys * (1.0 - case["masked"])
        side_q, side_k = b * lq * hq * d * size, keys * hk * d * size
        if not case["train"]:
            return {"bytes": 2 * side_q + 2 * side_k, "flops": 4.0 * seen * lq * hq * d}
        # q, dout, out, dq and k, v read; dk, dv written whole
        return {"bytes": 4 * side_q + 2 * side_k + 2 * b * lk * hk * d * size, "flops": 14.0 * seen * lq * hq * d}
    count = case["n"] * case["c"] * case["h"] * case["w"]
    maps = (4 if case["train"] else 2)
    if case["op"] == "norm":
        maps += (2 if case["train"] else 1) if case["residual"] else 0
        return {"bytes": maps * count * size + 16 * case["c"], "flops": (24.0 if case["train"] else 8.0) * count}
    # with a residual its gradient is the output's: nothing more to write
    return {"bytes": (maps + (1 if case["residual"] else 0)) * count * size, "flops": 4.0 * count}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, state)
    if case["op"] == "attention":
        return _exact_attention(case, state)
    return _exact_dropout(case, state)


def _exact_norm(case, s):
    """The definition, image by image; the gradients by differentiation of it."""
    ys, dxs, drs = [], [], []
    weight, bias = s["weight"].detach().double(), s["bias"].detach().double()
    if case["train"]:
        weight.requires_grad_(True)
        bias.requires_grad_(True)
    dw, db = torch.zeros_like(weight), torch.zeros_like(bias)
    for i in range(case["n"]):
        x = s["x"][i].detach().double()
        r = s["residual"][i].detach().double() if s["residual"] is not None else None
        wanted = [x] + ([r] if r is not None else [])
        if case["train"]:
            for t in wanted:
                t.requires_grad_(True)
        groups = x.reshape(case["groups"], -1)
        var, mean = torch.var_mean(groups, dim=1, keepdim=True, unbiased=False)
        z = ((groups - mean) * torch.rsqrt(var + _EPS)).reshape(x.shape) * weight[:, None, None] + bias[:, None, None]
        if r is not None:
            z = z + r
        y = {"relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t), "none": lambda t: t}[case["act"]](z)
        ys.append(y.detach())
        if case["train"]:
            grads = torch.autograd.grad(y, wanted + [weight, bias], s["dout"][i].double())
            dxs.append(grads[0])
            if r is not None:
                drs.append(grads[1])
            dw, db = dw + grads[-2], db + grads[-1]
    out = (torch.stack(ys),)
    if case["train"]:
        out += (torch.stack(dxs), dw.detach(), db.detach())
        if drs:
            out += (torch.stack(drs),)
    return out


def _exact_attention(case, s):
    """Image by image and head by head, over the keys that take part alone; the gradients by differentiation."""
    b, lq, lk, hq, hk, d = (case[k] for k in ("b", "lq", "lk", "heads", "kv_heads", "dim"))
    lengths = [int(t) for t in case["lengths"].split(",")] if case["lengths"] else [lk] * b
    out = torch.zeros((b, lq, hq, d), dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (s["q"], s["k"], s["v"])]
    for i in range(b):
        taken = torch.arange(lengths[i], device="cuda")
        if s["mask"] is not None:
            taken = taken[s["mask"][i, :lengths[i]]]
        if taken.numel() == 0:
            continue
        for j in range(hq):
            m = j // (hq // hk)
            q = s["q"][i, :, j].detach().double()
            k, v = (s[t][i, taken, m].detach().double() for t in ("k", "v"))
            if case["train"]:
                for t in (q, k, v):
                    t.requires_grad_(True)
            o = torch.softmax(q @ k.t() / math.sqrt(d), dim=1) @ v
            out[i, :, j] = o.detach()
            if case["train"]:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["dout"][i, :, j].double())
                grads[0][i, :, j] = gq
                grads[1][i, taken, m] += gk
                grads[2][i, taken, m] += gv
    return (out, *grads) if case["train"] else (out,)


def _exact_dropout(case, s):
    """The generator on 16-bit limbs: no product here passes 33 bits."""
    x = s["x"].detach()
    n, c, h, w = x.shape
    count = x.numel()
    key = int(s["seed"].item()) if case["device_seed"] else s["seed"]

    def product(t, m):                                          # (high, low) words of t * m
        t0, t1, m0, m1 = t % 65536, t // 65536, m % 65536, m // 65536
        low = t0 * m0
        mid = t1 * m0 + low // 65536
        mid2 = t0 * m1 + mid % 65536
        return t1 * m1 + mid // 65536 + mid2 // 65536, (mid2 % 65536) * 65536 + low % 65536

    block = torch.arange((count + 7) // 8, dtype=torch.int64, device="cuda")
    ctr = [block % 4294967296, block // 4294967296, torch.zeros_like(block), torch.zeros_like(block)]
    for i in range(10):
        ki, kj = (key % 4294967296 + i * _W0) % 4294967296, (key // 4294967296 + i * _W1) % 4294967296
        h0, l0 = product(ctr[0], _M0)
        h1, l1 = product(ctr[2], _M1)
        ctr = [torch.bitwise_xor(torch.bitwise_xor(h1, ctr[1]), torch.full_like(h1, ki)), l1,
               torch.bitwise_xor(torch.bitwise_xor(h0, ctr[3]), torch.full_like(h0, kj)), l0]
    bits = torch.empty((block.numel(), 8), dtype=torch.int64, device="cuda")
    for i in range(4):
        bits[:, 2 * i], bits[:, 2 * i + 1] = ctr[i] % 65536, ctr[i] // 65536
    limit = _threshold(case["p"])
    keep = (bits.flatten()[:count] >= limit).double().reshape(n, h, w, c).permute(0, 3, 1, 2)
    keep = keep * (65536.0 / (65536.0 - limit))
    y = x.double() * keep
    if s["residual"] is not None:
        y = y + s["residual"].detach().double()
    out = (y, s["dout"].double() * keep)
    return out + ((s["dout"].double(),) if s["residual"] is not None else ())
