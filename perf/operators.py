"""Cases for timing three operators that a Vision Transformer is trained and served with: differential attention, group
normalisation with an activation on channels-last maps, and the clipping of gradients by their global norm.

`run` computes a case in plain torch operations, or, where `own` is true, through vit_amd's operators:

    vit_amd.diff_attention(q, k, v, lam, lambda_init, key_lens=None, causal=False)
    vit_amd.group_norm(x, num_groups, weight, bias, eps, activation)
    vit_amd.clip_grad_norm_(parameters, max_norm)
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one new token of 8 requests against a padded cache of their earlier tokens, four query heads to a key head
        dict(name="diff_token", op="diff", type="bf16", batch=8, nq=1, nk=2048, heads=8, kv_heads=2, d=64, lens=True,
             causal=False, shared=False, train=False),
        # ViT-B/16 at 224 px, a serving batch: 196 patches and the class token, heads of 64 channels in two maps of 32
        dict(name="diff_b16_224", op="diff", type="bf16", batch=64, nq=197, nk=197, heads=12, kv_heads=12, d=32,
             lens=False, causal=False, shared=True, train=False),
        # ViT-S/16 at 384 px in training: 577 tokens, heads of 96 channels
        dict(name="diff_s16_384_train", op="diff", type="bf16", batch=16, nq=577, nk=577, heads=8, kv_heads=8, d=48,
             lens=False, causal=False, shared=True, train=True),
        # a long causal sequence in training, two query heads to a key head, heads of 128 channels
        dict(name="diff_long_train", op="diff", type="bf16", batch=2, nq=4096, nk=4096, heads=8, kv_heads=4, d=64,
             lens=False, causal=True, shared=False, train=True),
        # the fp32 mode in training, ViT-H/14's head size, a padded batch of images of several sizes
        dict(name="diff_f32_train", op="diff", type="f32", batch=4, nq=257, nk=257, heads=16, kv_heads=16, d=40,
             lens=True, causal=False, shared=False, train=True),
        # one image's 14 x 14 map on its way to the tokens: latency counts
        dict(name="gn_one_image", op="gn", type="bf16", batch=1, height=14, width=14, channels=512, groups=32, act="silu",
             affine=True, train=False),
        # the first stage of a convolutional stem at 224 px, a serving batch
        dict(name="gn_stem_56", op="gn", type="bf16", batch=64, height=56, width=56, channels=256, groups=32, act="relu",
             affine=True, train=False),
        # a later stage in training
        dict(name="gn_stem_28_train", op="gn", type="bf16", batch=32, height=28, width=28, channels=512, groups=32,
             act="gelu", affine=True, train=True),
        # an odd map and odd groups in the fp32 mode in training
        dict(name="gn_f32_odd_train", op="gn", type="f32", batch=3, height=97, width=61, channels=90, groups=9, act="silu",
             affine=True, train=True),
        # fine-tuning of a head and the last block: few tensors, two types, the bound in force
        dict(name="clip_head", op="clip", layout="list", tensors=14, elements=2_000_003, bf16_share=0.5, clips=True),
        # every gradient of ViT-S/16 in one communication bucket, late in training: the norm is under the bound
        dict(name="clip_s16", op="clip", layout="bucket", tensors=106, elements=49_560_000, bf16_share=0.0, clips=False),
        # every gradient of ViT-L/16, the bound in force
        dict(name="clip_l16", op="clip", layout="bucket", tensors=298, elements=304_330_000, bf16_share=0.0, clips=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["diff", "gn", "clip"])
    if op == "diff":
        kind = rng.choice(["token", "image", "image", "sequence"])
        kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
        group = rng.choice([1, 1, 2, 4]) if kv <= 8 else 1
        heads = kv * group
        type_ = rng.choice(["bf16", "bf16", "f32"])
        train = rng.random() < 0.5
        d = rng.choice([16, 24, 32, 32, 40, 48, 64, 64])
        if kind == "token":
            nq, nk, batch, causal = _log(rng, 1, 9), _log(rng, 16, 9000), _log(rng, 1, 16), rng.random() < 0.5
        elif kind == "image":
            nq = nk = _log(rng, 17, 800)
            batch, causal = _log(rng, 1, 48), False
        else:
            nq = nk = _log(rng, 300, 2500)
            batch, causal = rng.choice([1, 2]), True
        while batch > 1 and batch * heads * nq * nk * (10 if type_ == "f32" else 1) > 1.3e8:
            batch = (batch + 1) // 2
        return dict(op=op, type=type_, batch=batch, nq=nq, nk=nk, heads=heads, kv_heads=kv, d=d, lens=rng.random() < 0.4,
                    causal=causal, shared=rng.random() < 0.5, train=train)
    if op == "gn":
        groups = rng.choice([1, 3, 4, 8, 16, 32, 32])
        channels = groups * _log(rng, 1, max(2, 1024 // groups))
        height = _log(rng, 2, 112)
        width = max(2, int(height * rng.uniform(0.6, 1.7)))
        if height * width * (channels // groups) < 64:                          # a handful of values has no deviation to speak of
            height = width = 8
        batch = max(1, min(_log(rng, 1, 128), int(2.4e7 / (height * width * channels))))
        return dict(op=op, type=rng.choice(["bf16", "f32"]), batch=batch, height=height, width=width, channels=channels,
                    groups=groups, act=rng.choice(["none", "relu", "gelu", "silu"]), affine=rng.random() < 0.85,
                    train=rng.random() < 0.5)
    layout = rng.choice(["list", "bucket"])
    tensors = _log(rng, 1, 30) if layout == "list" else _log(rng, 8, 400)
    return dict(op=op, layout=layout, tensors=tensors, elements=_log(rng, 1_000, 6e7) + tensors,
                bf16_share=rng.choice([0.0, 0.0, 0.3, 1.0]), clips=rng.random() < 0.6)


# ---- inputs ------------------------------------------------------------------------------------

def _normal(gen, *shape, type_=torch.float32, scale=1.0, shift=0.0):
    return torch.randn(*shape, device=DEV, generator=gen).mul_(scale).add_(shift).to(type_)


def _tensor_sizes(case, seed):
    """Sizes of the gradients: weights of many sizes beside short vectors, as a model has them."""
    r = torch.Generator().manual_seed(17 + case["tensors"])                     # the model does not change with the seed
    n, total = case["tensors"], case["elements"]
    share = torch.where(torch.arange(n) % 2 == 0, torch.rand(n, generator=r) + 0.1, torch.full((n,), 2e-4))
    sizes = (share / share.sum() * (total - n)).long() + 1
    sizes[0] += total - int(sizes.sum())
    return [int(s) for s in sizes]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    state = dict(case)
    if case["op"] == "diff":
        t, B, H, K, d = TYPES[case["type"]], case["batch"], case["heads"], case["kv_heads"], case["d"]
        # head-major, as the framework's fused projection writes them; the operator takes token-major views
        q = _normal(gen, B, H, case["nq"], 2, d, type_=t).permute(0, 2, 1, 3, 4)
        k = _normal(gen, B, K, case["nk"], 2, d, type_=t).permute(0, 2, 1, 3, 4)
        v = _normal(gen, B, K, case["nk"], 2 * d, type_=t).permute(0, 2, 1, 3)
        lam = _normal(gen, 4, d, scale=0.1) if case["shared"] else _normal(gen, 4, H, d, scale=0.1)
        state.update(q=q, k=k, v=v, lam=lam, lambda_init=0.8 - 0.6 * math.exp(-0.3 * 4), key_lens=None)
        if case["lens"]:
            nk = case["nk"]
            lens = torch.randint(max(1, nk // 3), nk + 1, (B,), device=DEV, generator=gen, dtype=torch.int32)
            lens[0] = nk
            state["key_lens"] = lens
        if case["train"]:
            for n in ("q", "k", "v", "lam"):
                state[n].requires_grad_(True)
            state["dout"] = _normal(gen, B, case["nq"], H, 2 * d, type_=t)
    elif case["op"] == "gn":
        t, C = TYPES[case["type"]], case["channels"]
        shape = (case["batch"], case["height"], case["width"], C)
        state["x"] = _normal(gen, *shape, type_=t, scale=1.5, shift=0.4)
        state["weight"] = _normal(gen, C, scale=0.2, shift=1.0) if case["affine"] else None
        state["bias"] = _normal(gen, C, scale=0.2) if case["affine"] else None
        if case["train"]:
            for n in ("x", "weight", "bias"):
                if state[n] is not None:
                    state[n].requires_grad_(True)
            state["dout"] = _normal(gen, *shape, type_=t)
    else:
        sizes = _tensor_sizes(case, seed)
        first16 = len(sizes) - int(round(case["bf16_share"] * len(sizes)))
        types = [torch.float32] * first16 + [torch.bfloat16] * (len(sizes) - first16)
        if case["layout"] == "list":
            grads = [_normal(gen, s, type_=t, scale=1e-2) for s, t in zip(sizes, types)]
            state["buffers"] = grads
        else:
            state["buffers"], grads = [], []
            for t in (torch.float32, torch.bfloat16):
                part = [s for s, u in zip(sizes, types) if u == t]
                if part:
                    flat = _normal(gen, sum(part), type_=t, scale=1e-2)
                    state["buffers"].append(flat)
                    grads += list(flat.split(part))                              # odd offsets, as in a bucket
        norm = 1e-2 * math.sqrt(sum(sizes))
        state["params"] = [g.detach() for g in grads]                            # only their .grad is looked at
        for p, g in zip(state["params"], grads):
            p.grad = g
        state["max_norm"] = 0.37 * norm if case["clips"] else 4.0 * norm
        state["tighten"] = 1.0 - 2.0 ** -11 if case["clips"] else 1.0
    return state


# ---- one pass ----------------------------------------------------------------------------------

def _visible(s):
    """[batch or 1, 1, 1, 1, nq, nk] truth values: which keys a query sees, or None for all of them."""
    nq, nk, seen = s["nq"], s["nk"], None
    cols = torch.arange(nk, device=DEV)
    if s["key_lens"] is not None:
        seen = (cols < s["key_lens"][:, None]).view(-1, 1, 1, 1, 1, nk)
    if s["causal"]:
        past = (cols[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)).view(1, 1, 1, 1, nq, nk)
        seen = past if seen is None else seen & past
    return seen


def _plain_diff(s, q, k, v, lam):
    B, nq, nk, H, K, d = s["batch"], s["nq"], s["nk"], s["heads"], s["kv_heads"], s["d"]
    q = q.permute(0, 2, 3, 1, 4).reshape(B, K, H // K, 2, nq, d)
    k = k.permute(0, 2, 3, 4, 1).reshape(B, K, 1, 2, d, nk)
    scores = q @ k * d ** -0.5
    seen = _visible(s)
    if seen is None:
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
    else:
        top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
        p = (scores - top.masked_fill(top == -math.inf, 0.0)).masked_fill(~seen, -math.inf).exp()
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    dots = (lam[0::2] * lam[1::2]).sum(-1).exp()                                # [2] or [2, heads]
    weight = (dots[0] - dots[1] + s["lambda_init"]).expand(H).reshape(1, K, H // K, 1, 1)
    p = p[:, :, :, 0] - weight * p[:, :, :, 1]
    out = p @ v.permute(0, 2, 1, 3).unsqueeze(2)                                # [B, K, H / K, nq, 2 d]
    return out.reshape(B, H, nq, 2 * d).permute(0, 2, 1, 3)


def _plain_gn(s, x, weight, bias):
    B, C, G = s["batch"], s["channels"], s["groups"]
    y = x.reshape(B, -1, G, C // G)
    mean = y.mean((1, 3), keepdim=True)
    y = y - mean
    y = (y * (y.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()).reshape(x.shape)
    if weight is not None:
        y = y * weight + bias
    if s["act"] == "relu":
        return y.clamp(min=0.0)
    if s["act"] == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))
    if s["act"] == "silu":
        return y / (1.0 + (-y).exp())
    return y


def _plain_clip(s):
    squares = torch.stack([b.double().square().sum() for b in s["buffers"]])
    norm = squares.sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return norm.float(), [b.copy_(b.float() * coef) for b in s["buffers"]]


def _step(s, names, plain, fused):
    """The operator's output, and in training the gradients of what requires them."""
    ins = [s[n] for n in names]
    if not s["train"]:
        with torch.no_grad():
            if own:
                return fused(*ins)
            return plain(s, *[None if t is None else t.float() for t in ins]).to(ins[0].dtype)
    live = [t for t in ins if t is not None]
    if own:
        out = fused(*ins)
        return [out] + list(torch.autograd.grad(out, live, s["dout"]))
    wide = [None if t is None else t.detach().float().requires_grad_(True) for t in ins]
    out = plain(s, *wide)
    grads = torch.autograd.grad(out, [t for t in wide if t is not None], s["dout"].float())
    return [out.detach().to(ins[0].dtype)] + [g.to(t.dtype) for g, t in zip(grads, live)]


def run(state):
    s = state
    if own:
        import vit_amd
    if s["op"] == "diff":
        return _step(s, ("q", "k", "v", "lam"), _plain_diff,
                     lambda q, k, v, lam: vit_amd.diff_attention(q, k, v, lam, s["lambda_init"], key_lens=s["key_lens"],
                                                                 causal=s["causal"]))
    if s["op"] == "gn":
        return _step(s, ("x", "weight", "bias"), _plain_gn,
                     lambda x, w, b: vit_amd.group_norm(x, s["groups"], w, b, 1e-5, s["act"]))
    # the bound tightens a little from step to step, so that a pass clips what the pass before it has clipped
    if own:
        norm, buffers = vit_amd.clip_grad_norm_(s["params"], s["max_norm"]), s["buffers"]
    else:
        norm, buffers = _plain_clip(s)
    s["max_norm"] *= s["tighten"]
    return [norm] + list(buffers)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    if case["op"] == "diff":
        B, nq, nk, H, K, d = (case[n] for n in ("batch", "nq", "nk", "heads", "kv_heads", "d"))
        size = 2 if case["type"] == "bf16" else 4
        lens = nk
        if case["lens"]:                                                       # the mean of the drawn lengths
            lens = (nk + (B - 1) * (max(1, nk // 3) + nk) / 2) / B
        q, kv = B * nq * H * 2 * d * size, B * lens * K * 4 * d * size
        pairs = B * H * nq * lens
        if case["causal"] and not case["lens"]:
            first = max(0, nk - nq)
            pairs = B * H * sum(range(first + 1, nk + 1)) if nq <= nk else B * H * nk * (nk + 1) // 2
        if not case["train"]:
            return {"bytes": 2 * q + kv, "flops": pairs * 8 * d}               # scores of two maps, one product with V
        # backward: scores again, dO V^T, dV, dQ and dK of two maps
        return {"bytes": 5 * q + 3 * kv, "flops": pairs * (8 + 20) * d}
    if case["op"] == "gn":
        n = case["batch"] * case["height"] * case["width"] * case["channels"] * (2 if case["type"] == "bf16" else 4)
        return {"bytes": (5 if case["train"] else 2) * n, "flops": 0}
    wide = 4 - 2 * case["bf16_share"]
    return {"bytes": case["elements"] * wide * (3 if case["clips"] else 1), "flops": 0}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _exact_diff(s):
    B, H, K, d, train = s["batch"], s["heads"], s["kv_heads"], s["d"], s["train"]
    q, k, v, lam = (s[n].detach().double() for n in ("q", "k", "v", "lam"))
    nq, nk = q.shape[1], k.shape[1]
    lam = lam if lam.dim() == 3 else lam[:, None].expand(4, H, d)
    e1, e2 = (lam[0] * lam[1]).sum(-1).exp(), (lam[2] * lam[3]).sum(-1).exp()
    out = torch.zeros(B, nq, H, 2 * d, dtype=torch.float64, device=DEV)
    dq, dk, dv, dlam, dw = (torch.zeros_like(t) for t in (q, k, v, lam, e1))
    for b in range(B):
        n = nk if s["key_lens"] is None else int(s["key_lens"][b])
        hidden = None
        if s["causal"]:
            hidden = torch.ones(nq, n, dtype=torch.bool, device=DEV).triu(nk - nq + 1)
        for h in range(H):
            g, w = h // (H // K), float(e1[h] - e2[h]) + s["lambda_init"]
            maps = []
            for m in (0, 1):
                a = q[b, :, h, m] @ k[b, :n, g, m].T / math.sqrt(d)
                if hidden is not None:
                    a = a.masked_fill(hidden, -math.inf)
                maps.append(torch.softmax(a, -1).nan_to_num(0.0))               # a row without keys is 0
            both = maps[0] - w * maps[1]
            out[b, :, h] = both @ v[b, :n, g]
            if not train:
                continue
            go = s["dout"][b, :, h].double()
            dv[b, :n, g] += both.T @ go
            da = go @ v[b, :n, g].T
            for m, c in ((0, 1.0), (1, -w)):
                mean = (maps[m] * da).sum(-1, keepdim=True)
                ds = c * maps[m] * (da - mean) / math.sqrt(d)
                dq[b, :, h, m] = ds @ k[b, :n, g, m]
                dk[b, :n, g, m] += ds.T @ q[b, :, h, m]
                if m == 1:
                    dw[h] -= mean.sum()
    if not train:
        return out
    for i, e, sign in ((0, e1, 1.0), (2, e2, -1.0)):
        dlam[i] = sign * (dw * e)[:, None] * lam[i + 1]
        dlam[i + 1] = sign * (dw * e)[:, None] * lam[i]
    return [out, dq, dk, dv, dlam if s["lam"].dim() == 3 else dlam.sum(1)]


def _exact_gn(s):
    x, G, train = s["x"].detach().double(), s["groups"], s["train"]
    C = x.shape[-1]
    one = torch.ones(C, dtype=torch.float64, device=DEV)
    w = one if s["weight"] is None else s["weight"].detach().double()
    b = 0 * one if s["bias"] is None else s["bias"].detach().double()
    g = x.unflatten(-1, (G, C // G))
    var, mean = torch.var_mean(g, (1, 2, 4), correction=0, keepdim=True)
    hat = (g - mean) / torch.sqrt(var + 1e-5)
    z = hat.flatten(-2) * w + b
    if s["act"] == "relu":
        out, slope = torch.relu(z), (z > 0).double()
    elif s["act"] == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        out, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif s["act"] == "silu":
        cdf = torch.sigmoid(z)
        out, slope = z * cdf, cdf * (1 + z * (1 - cdf))
    else:
        out, slope = z, torch.ones_like(z)
    if not train:
        return out
    dz = s["dout"].double() * slope
    dh = (dz * w).unflatten(-1, (G, C // G))
    dx = (dh - dh.mean((1, 2, 4), keepdim=True) - hat * (dh * hat).mean((1, 2, 4), keepdim=True)) / torch.sqrt(var + 1e-5)
    if s["weight"] is None:
        return [out, dx.flatten(-2)]
    return [out, dx.flatten(-2), (dz * hat.flatten(-2)).sum((0, 1, 2)), dz.sum((0, 1, 2))]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "diff":
        return _exact_diff(s)
    if case["op"] == "gn":
        return _exact_gn(s)
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(b, dtype=torch.float64)) ** 2 for b in s["buffers"]))
    c = min(1.0, s["max_norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64)] + [b.double() * c for b in s["buffers"]]
