"""Cases of the transformer layer's attention-side operators and their plain forms.

* ``attention``: grouped-query softmax attention with its recomputing backward
  (``transformer.functional.fused_grouped_attention``);
* ``qk_norm_rope``: RMS norm of every query / key head and the rotary position embedding in one pass
  (``transformer.functional.fused_qk_norm_rope``);
* ``dropout``: counter-based dropout whose mask is never stored (``transformer.functional.fused_dropout``).

Tensors are in this package's [sequence, batch, heads, head_dim] layout; query, key and value are views of
one fused projection output, as the transformer layer has them.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_M32 = 0xFFFFFFFF


def listed():
    return [
        # one new token for each of 8 sequences against caches of unequal lengths (latency of one decode step)
        {"name": "attn_decode", "op": "attention", "dt": "bf16", "sq": 1, "sk": 4099, "b": 8, "np": 32, "ng": 8, "hn": 128,
         "causal": True, "window": 0, "lens": True, "p": 0.0, "train": False},
        # a small ragged training step: odd length, a head size that fills no tile, padded batch with an empty sequence
        {"name": "attn_odd_train", "op": "attention", "dt": "fp16", "sq": 193, "sk": 193, "b": 3, "np": 6, "ng": 2, "hn": 80,
         "causal": True, "window": 0, "lens": True, "p": 0.0, "train": True},
        # GPT-2-medium's training attention: 8 x 1024 tokens, 16 heads of 64, attention dropout 0.1
        {"name": "attn_gpt2_train", "op": "attention", "dt": "bf16", "sq": 1024, "sk": 1024, "b": 8, "np": 16, "ng": 16, "hn": 64,
         "causal": True, "window": 0, "lens": False, "p": 0.1, "train": True},
        # sliding-window training step
        {"name": "attn_window_train", "op": "attention", "dt": "fp16", "sq": 4096, "sk": 4096, "b": 2, "np": 16, "ng": 4, "hn": 128,
         "causal": True, "window": 512, "lens": False, "p": 0.0, "train": True},
        # long-context training step, four query heads to a key head
        {"name": "attn_long_train", "op": "attention", "dt": "bf16", "sq": 8192, "sk": 8192, "b": 1, "np": 32, "ng": 8, "hn": 128,
         "causal": True, "window": 0, "lens": False, "p": 0.0, "train": True},
        # encoder / cross attention without a causal mask, forward only (evaluation)
        {"name": "attn_full_eval", "op": "attention", "dt": "bf16", "sq": 2048, "sk": 2500, "b": 4, "np": 16, "ng": 16, "hn": 128,
         "causal": False, "window": 0, "lens": False, "p": 0.0, "train": False},
        # one decode step of 16 sequences: every token at a position of its own
        {"name": "rope_decode", "op": "qk_norm_rope", "dt": "bf16", "s": 1, "b": 16, "np": 32, "ng": 8, "hn": 128, "rot": 128,
         "inter": False, "norm": True, "pos": True, "train": False},
        # GPT-2-medium's shapes with a norm and rotation added, training
        {"name": "rope_gpt2_train", "op": "qk_norm_rope", "dt": "bf16", "s": 1024, "b": 8, "np": 16, "ng": 16, "hn": 64, "rot": 64,
         "inter": False, "norm": True, "pos": False, "train": True},
        # partial interleaved rotation in fp32 at odd sizes, training
        {"name": "rope_odd_fp32", "op": "qk_norm_rope", "dt": "fp32", "s": 777, "b": 3, "np": 6, "ng": 2, "hn": 80, "rot": 20,
         "inter": True, "norm": True, "pos": True, "train": True},
        # long-context training step
        {"name": "rope_long_train", "op": "qk_norm_rope", "dt": "bf16", "s": 8192, "b": 2, "np": 32, "ng": 8, "hn": 128, "rot": 128,
         "inter": False, "norm": True, "pos": False, "train": True},
        # embedding dropout of GPT-2-medium, forward and backward
        {"name": "drop_embedding", "op": "dropout", "dt": "bf16", "shape": "1024,8,1024", "p": 0.1},
        # dropout of an odd number of fp32 activations, largest
        {"name": "drop_large_fp32", "op": "dropout", "dt": "fp32", "shape": "8191,3,4099", "p": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "qk_norm_rope", "dropout"])
    dt = rng.choice(["bf16", "fp16"])
    if op == "attention":
        hn = rng.choice([40, 64, 64, 80, 96, 128, 128])
        ng, r = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        train = rng.random() < 0.6
        sk = _log(rng, 1, 6000)
        sq = sk if train or rng.random() < 0.3 else min(sk, _log(rng, 1, 600)) if rng.random() < 0.8 else _log(rng, 1, 2000)
        while sq * sk * ng * r > 2 ** 29 and ng * r > 1:  # at most a quarter of the scores of the largest listed case
            ng, r = (ng // 2, r) if ng > 1 else (ng, r - 1)
        b = max(1, min(_log(rng, 1, 32), int(2 ** 28 / max(1, sq * sk * ng * r)), 2 ** 17 // sk + 1))
        causal = rng.random() < 0.7
        return {"op": op, "dt": dt, "sq": sq, "sk": sk, "b": b, "np": ng * r, "ng": ng, "hn": hn, "causal": causal,
                "window": _log(rng, 1, sk) if causal and rng.random() < 0.3 else 0, "lens": rng.random() < 0.4,
                "p": rng.choice([0.0, 0.0, 0.1, 0.3]) if train else 0.0, "train": train}
    if op == "qk_norm_rope":
        hn = rng.choice([64, 80, 96, 128, 128, 256])
        ng, r = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4])
        s = min(_log(rng, 1, 9000), int(3e7 / (ng * r * hn)))
        b = max(1, min(_log(rng, 1, 32), int(3e7 / (s * ng * r * hn))))
        return {"op": op, "dt": rng.choice(["bf16", "fp16", "fp32"]), "s": s, "b": b, "np": ng * r, "ng": ng, "hn": hn,
                "rot": rng.choice([hn, hn, hn // 2, hn // 4]), "inter": rng.random() < 0.4, "norm": rng.random() < 0.8,
                "pos": rng.random() < 0.5, "train": rng.random() < 0.7}
    return {"op": op, "dt": rng.choice(["bf16", "fp16", "fp32"]),
            "shape": "%d,%d,%d" % (_log(rng, 1, 4000), rng.randint(1, 8), _log(rng, 1, 3000)),
            "p": rng.choice([0.05, 0.1, 0.25, 0.5, 0.9])}


def _attention_pairs(c):
    """Unmasked (query, key) pairs of one head of a full-length sequence."""
    sq, sk = c["sq"], c["sk"]
    if not c["causal"]:
        return sq * sk
    n = 0
    off = sk - sq
    w = c["window"] or sk
    # query i sees keys max(0, i + off - w + 1) .. i + off
    for i in range(sq):
        n += max(0, i + off + 1 - max(0, i + off - w + 1))
    return n


def work(case):
    c = case
    if c["op"] == "attention":
        q, kv = c["sq"] * c["b"] * c["np"] * c["hn"], c["sk"] * c["b"] * c["ng"] * c["hn"]
        pairs = _attention_pairs(c) * c["b"] * c["np"]
        if c["lens"]:  # key lengths are spread evenly over 0 .. sk: about half of the keys are there
            pairs, kv = pairs // 2, kv // 2
        el = 2
        if not c["train"]:
            return {"bytes": el * (2 * q + 2 * kv), "flops": 4 * pairs * c["hn"]}
        return {"bytes": el * (4 * q + 4 * kv), "flops": 14 * pairs * c["hn"]}
    el = 4 if c["dt"] == "fp32" else 2
    if c["op"] == "qk_norm_rope":
        n = c["s"] * c["b"] * (c["np"] + c["ng"]) * c["hn"]
        return {"bytes": el * n * (4 if c["train"] else 2), "flops": n * (24 if c["train"] else 8)}
    n = math.prod(int(x) for x in c["shape"].split(","))
    return {"bytes": el * n * 4, "flops": n * 20}


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dt"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    st = {"c": c}
    if c["op"] == "attention":
        sq, sk, b, np_, ng, hn = c["sq"], c["sk"], c["b"], c["np"], c["ng"], c["hn"]
        if sq == sk:  # views of the fused projection output
            mixed = randn(sq, b, (np_ + 2 * ng) * hn).to(dt)
            q = mixed[..., :np_ * hn].view(sq, b, np_, hn)
            k = mixed[..., np_ * hn:(np_ + ng) * hn].view(sk, b, ng, hn)
            v = mixed[..., (np_ + ng) * hn:].view(sk, b, ng, hn)
        else:
            kv = randn(sk, b, 2 * ng * hn).to(dt)
            q = randn(sq, b, np_, hn).to(dt)
            k, v = kv[..., :ng * hn].view(sk, b, ng, hn), kv[..., ng * hn:].view(sk, b, ng, hn)
        st["q"], st["k"], st["v"] = (t.detach().requires_grad_(c["train"]) for t in (q, k, v))
        st["dout"] = randn(sq, b, np_, hn).to(dt) if c["train"] else None
        if c["lens"]:  # unequal lengths, evenly spread; an empty sequence where the batch is larger than one
            lens = torch.linspace(0 if b > 1 else sk, sk, b, device="cuda").round().to(torch.int32)
            st["lens"] = lens[torch.randperm(b, device="cuda", generator=g)].contiguous()
        else:
            st["lens"] = None
        st["seed"] = int(torch.randint(1 << 62, (1,), device="cuda", generator=g).item())
        return st
    if c["op"] == "qk_norm_rope":
        s, b, np_, ng, hn = c["s"], c["b"], c["np"], c["ng"], c["hn"]
        mixed = randn(s, b, (np_ + 2 * ng) * hn).to(dt)
        train = c["train"]
        st["q"] = mixed[..., :np_ * hn].view(s, b, np_, hn).detach().requires_grad_(train)
        st["k"] = mixed[..., np_ * hn:(np_ + ng) * hn].view(s, b, ng, hn).detach().requires_grad_(train)
        st["wq"] = st["wk"] = None
        if c["norm"]:
            st["wq"] = (1 + 0.2 * randn(hn)).requires_grad_(train)
            st["wk"] = (1 + 0.2 * randn(hn)).requires_grad_(train)
        n_pos = 16384
        ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["pos"] = torch.randint(n_pos, (s, b), device="cuda", generator=g) if c["pos"] else None
        st["dq"], st["dk"] = (randn(s, b, np_, hn).to(dt), randn(s, b, ng, hn).to(dt)) if train else (None, None)
        return st
    shape = [int(x) for x in c["shape"].split(",")]
    st["x"] = randn(*shape).to(dt).requires_grad_(True)
    st["dy"] = randn(*shape).to(dt)
    st["seed"] = int(torch.randint(1 << 62, (1,), device="cuda", generator=g).item())
    return st


# ---- plain forms -----------------------------------------------------------------------------------------

def _mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & _M32
    return x ^ (x >> 16)


def _attention_keep(seed, bh, sq, sk, p, dev):
    """Keep flags [bh, sq, sk] of attention dropout: a hash of (seed, head, query), then one of (that, key pair),
    whose low and high half decide about the even and the odd key."""
    lo, hi = seed & _M32, (seed >> 32) & _M32
    h = (torch.arange(bh, device=dev) * 0x9E3779B1)[:, None] & _M32
    q = (torch.arange(sq, device=dev) * 0x85EBCA77)[None] & _M32
    row = _mix32(lo ^ _mix32(hi ^ h ^ q))
    pair = (torch.arange((sk + 1) // 2, device=dev) * 0x9E3779B9) & _M32
    x = (row[..., None] + pair) & _M32
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 16)
    t = min(65536, int((1.0 - p) * 65536.0))
    return torch.stack(((x & 0xFFFF) < t, (x >> 16) < t), -1).flatten(-2)[..., :sk]


def _attention_allowed(c, lens, dev):
    """Whether a query sees a key: [1 or b, 1, sq, sk]."""
    sq, sk = c["sq"], c["sk"]
    i = torch.arange(sq, device=dev)[:, None] + (sk - sq)
    j = torch.arange(sk, device=dev)[None]
    ok = torch.ones(sq, sk, dtype=torch.bool, device=dev)
    if c["causal"]:
        ok = ok & (j <= i)
        if c["window"]:
            ok = ok & (j > i - c["window"])
    ok = ok[None, None]
    return ok if lens is None else ok & (j < lens.view(-1, 1, 1, 1))


def _attention_plain(st):
    c = st["c"]
    sq, sk, b, np_, ng, hn = c["sq"], c["sk"], c["b"], c["np"], c["ng"], c["hn"]
    r, scale, dev = np_ // ng, hn ** -0.5, st["q"].device
    dt = st["q"].dtype
    # [b, ng, r * sq, hn] and [b, ng, sk, hn]: the heads of a group share their keys in one product
    q = st["q"].detach().float().view(sq, b, ng, r, hn).permute(1, 2, 3, 0, 4).reshape(b, ng, r * sq, hn)
    k = st["k"].detach().float().permute(1, 2, 0, 3).contiguous()
    v = st["v"].detach().float().permute(1, 2, 0, 3).contiguous()
    ok = _attention_allowed(c, st["lens"], dev).repeat(1, 1, r, 1)
    s = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    prob = s.sub_(m).exp_()
    prob = prob.div_(prob.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny))
    keep = None
    if c["p"] > 0:
        keep = _attention_keep(st["seed"], b * np_, sq, sk, c["p"], dev).view(b, ng, r * sq, sk).float() / (1 - c["p"])
    dropped = prob if keep is None else prob * keep
    out = dropped @ v

    def queries(t):
        return t.view(b, ng, r, sq, hn).permute(3, 0, 1, 2, 4).reshape(sq, b, np_, hn).to(dt)

    if not c["train"]:
        return (queries(out),)
    do = st["dout"].float().view(sq, b, ng, r, hn).permute(1, 2, 3, 0, 4).reshape(b, ng, r * sq, hn)
    dv = dropped.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    if keep is not None:
        dp = dp.mul_(keep)
    ds = dp.sub_((prob * dp).sum(-1, keepdim=True)).mul_(prob).mul_(scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    return queries(out), queries(dq), dk.permute(2, 0, 1, 3).to(dt), dv.permute(2, 0, 1, 3).to(dt)


def _rotate(x, cos, sin, inter, sign):
    """Rotates the first 2 * cos.size(-1) values of the last axis by sign * angle."""
    h = cos.size(-1)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if inter else (x[..., :h], x[..., h:2 * h])
    y, z = a * cos - sign * b * sin, b * cos + sign * a * sin
    yz = torch.stack((y, z), -1).flatten(-2) if inter else torch.cat((y, z), -1)
    return torch.cat((yz, x[..., 2 * h:]), -1)


def _norm_rope_plain(st):
    c = st["c"]
    if st["pos"] is None:
        cos, sin = st["cos"][:c["s"], None, None], st["sin"][:c["s"], None, None]
    else:
        cos, sin = st["cos"][st["pos"]][:, :, None], st["sin"][st["pos"]][:, :, None]
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st["dq"]), (st["k"], st["wk"], st["dk"])):
        dt, x = x.dtype, x.detach().float()
        n = x
        if w is not None:
            w = w.detach()
            rs = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            n = x * rs * w
        outs.append(_rotate(n, cos, sin, c["inter"], 1.0).to(dt))
        if not c["train"]:
            continue
        dn = _rotate(dy.float(), cos, sin, c["inter"], -1.0)
        if w is None:
            grads.append(dn.to(dt))
            continue
        xh, gw = x * rs, dn * w
        wgrads.append((dn * xh).double().sum((0, 1, 2)).float())
        grads.append((rs * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(dt))
    return (*outs, *grads, *wgrads)


def _philox_keep(seed, n, p, dev):
    """Keep flags [n]: Philox4x32-7 of (element // 4) under the key `seed`, word element % 4, against (1 - p) 2^32."""
    calls = torch.arange((n + 3) // 4, device=dev)
    c0, c1 = calls & _M32, calls >> 32
    c2, c3 = torch.zeros_like(calls), torch.zeros_like(calls)
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(7):  # the seven rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    t = min(_M32, int((1.0 - p) * 4294967296.0))
    return (torch.stack((c0, c1, c2, c3), -1).flatten()[:n]) < t


def _dropout_plain(st):
    c = st["c"]
    x, dy = st["x"].detach(), st["dy"]
    keep = _philox_keep(st["seed"], x.numel(), c["p"], x.device).view(x.shape)
    inv = 1.0 / (1.0 - c["p"])
    zero = torch.zeros((), device=x.device)
    return torch.where(keep, x.float() * inv, zero).to(x.dtype), torch.where(keep, dy.float() * inv, zero).to(x.dtype)


# ---- the framework's calls -------------------------------------------------------------------------------

def _attention_own(st):
    from beforeholiday_amd.transformer.functional import fused_grouped_attention

    c = st["c"]
    out = fused_grouped_attention(st["q"], st["k"], st["v"], causal=c["causal"], window=c["window"] or None,
                                  key_lengths=st["lens"], dropout_p=c["p"], training=c["train"], seed=st["seed"])
    if not c["train"]:
        return (out,)
    return (out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"]))


def _norm_rope_own(st):
    from beforeholiday_amd.transformer.functional import fused_qk_norm_rope

    c = st["c"]
    q, k = fused_qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], positions=st["pos"],
                              interleaved=c["inter"])
    if not c["train"]:
        return q, k
    leaves = (st["q"], st["k"]) + ((st["wq"], st["wk"]) if c["norm"] else ())
    return (q, k, *torch.autograd.grad((q, k), leaves, (st["dq"], st["dk"])))


def _dropout_own(st):
    from beforeholiday_amd.transformer.functional import fused_dropout

    y = fused_dropout(st["x"], st["c"]["p"], True, seed=st["seed"])
    return (y, *torch.autograd.grad(y, st["x"], st["dy"]))


def run(state):
    op = state["c"]["op"]
    if own:
        return {"attention": _attention_own, "qk_norm_rope": _norm_rope_own, "dropout": _dropout_own}[op](state)
    return {"attention": _attention_plain, "qk_norm_rope": _norm_rope_plain, "dropout": _dropout_plain}[op](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------

def _exact_attention(st):
    c = st["c"]
    sq, sk, b, np_, ng, hn = c["sq"], c["sk"], c["b"], c["np"], c["ng"], c["hn"]
    if b * np_ > 4096:
        return None
    r, dev = np_ // ng, st["q"].device
    f8 = torch.float64
    out, dq = (torch.zeros(sq, b, np_, hn, dtype=f8, device=dev) for _ in range(2))
    dk, dv = (torch.zeros(sk, b, ng, hn, dtype=f8, device=dev) for _ in range(2))
    lens = [sk] * b if st["lens"] is None else st["lens"].tolist()
    rows = torch.arange(sq, device=dev)
    step = max(1, (1 << 26) // max(1, sk))  # queries of one head at a time
    for n in range(b):
        for h in range(np_):
            k, v = (st[x][:, n, h // r].detach().to(f8) for x in "kv")
            for i0 in range(0, sq, step):
                q = st["q"][i0:i0 + step, n, h].detach().to(f8)
                at = rows[i0:i0 + step].unsqueeze(1) + (sk - sq)
                key = torch.arange(sk, device=dev).unsqueeze(0)
                see = (key < lens[n]).expand(q.size(0), sk)
                if c["causal"]:
                    see = see & (at >= key)
                if c["window"]:
                    see = see & (at - key < c["window"])
                z = (q @ k.t()) / math.sqrt(hn)
                e = torch.exp(z - torch.where(see, z, -1e300).max(1, keepdim=True).values) * see
                tot = e.sum(1, keepdim=True)
                a = torch.where(tot > 0, e / torch.where(tot > 0, tot, 1.0), 0.0)
                w = torch.ones_like(a)
                if c["p"] > 0:
                    w = _exact_keep(st["seed"], n * np_ + h, rows[i0:i0 + step], sk, c["p"]).to(f8) / (1.0 - c["p"])
                out[i0:i0 + step, n, h] = (a * w) @ v
                if c["train"]:
                    g = st["dout"][i0:i0 + step, n, h].to(f8)
                    dv[:, n, h // r] += (a * w).t() @ g
                    da = (g @ v.t()) * w
                    dz = a * (da - (a * da).sum(1, keepdim=True)) / math.sqrt(hn)
                    dq[i0:i0 + step, n, h] = dz @ k
                    dk[:, n, h // r] += dz.t() @ q
    return (out, dq, dk, dv) if c["train"] else (out,)


def _exact_keep(seed, head, rows, sk, p):
    """The dropout decisions of one head's rows, key by key."""
    def avalanche(x):
        for shift, mul in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            x = ((x ^ (x >> shift)) * mul) % (1 << 32)
        return x ^ (x >> 16)
    inner = avalanche((rows * 0x85EBCA77) % (1 << 32) ^ (head * 0x9E3779B1) % (1 << 32) ^ (seed >> 32))
    base = avalanche(inner ^ (seed % (1 << 32)))
    key = torch.arange(sk, device=rows.device)
    x = (base[:, None] + (key // 2) * 0x9E3779B9) % (1 << 32)
    x = (x ^ (x >> 16)) * 0x7FEB352D % (1 << 32)
    x = x ^ (x >> 16)
    return torch.where(key % 2 == 1, x // 65536, x % 65536) < min(65536, math.floor((1.0 - p) * 65536))


def _exact_norm_rope(st):
    c = st["c"]
    h, f8 = c["rot"] // 2, torch.float64
    first = torch.arange(h, device="cuda") * 2 if c["inter"] else torch.arange(h, device="cuda")
    second = first + (1 if c["inter"] else h)
    pos = torch.arange(c["s"], device="cuda")[:, None].expand(-1, c["b"]) if st["pos"] is None else st["pos"]
    # the rotation as a unit complex number for each position; the tables are the operator's inputs
    turn = torch.complex(st["cos"].to(f8), st["sin"].to(f8))[pos][:, :, None]
    ys, gs, ws = [], [], []
    for name, wname, dname in (("q", "wq", "dq"), ("k", "wk", "dk")):
        x = st[name].detach().to(f8)
        w = None if st[wname] is None else st[wname].detach().to(f8)
        n = x
        if w is not None:
            length = torch.sqrt(x.square().sum(-1, keepdim=True) / c["hn"] + 1e-6)
            n = x / length * w
        y = n.clone()
        z = torch.complex(n[..., first], n[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        ys.append(y)
        if c["train"]:
            d = st[dname].to(f8)
            t = d.clone()
            z = torch.complex(d[..., first], d[..., second]) * turn.conj()
            t[..., first], t[..., second] = z.real, z.imag
            if w is None:
                gs.append(t)
            else:
                ws.append((t * x / length).flatten(0, 2).sum(0))
                along = (t * w * x).sum(-1, keepdim=True)
                gs.append(t * w / length - x * along / (c["hn"] * length ** 3))
    return (*ys, *gs, *ws)


def _exact_dropout(st):
    n, dev = st["x"].numel(), st["x"].device
    key = [st["seed"] % (1 << 32), st["seed"] >> 32]
    i = torch.arange((n + 3) // 4, device=dev)
    ctr = [i % (1 << 32), i // (1 << 32), i * 0, i * 0]

    def halves(a, m):  # a * m for a < 2^32, m < 2^32 as (high, low) 32-bit words, by 16-bit parts
        lo, hi = (a % 65536) * m, (a // 65536) * m
        mid = hi + lo // 65536
        return mid // 65536, (mid % 65536) * 65536 + lo % 65536
    for k in range(7):
        h0, l0 = halves(ctr[0], 0xD2511F53)
        h1, l1 = halves(ctr[2], 0xCD9E8D57)
        a, b = (key[0] + k * 0x9E3779B9) % (1 << 32), (key[1] + k * 0xBB67AE85) % (1 << 32)
        ctr = [h1 ^ ctr[1] ^ a, l1, h0 ^ ctr[3] ^ b, l0]
    p = st["c"]["p"]
    stay = torch.stack(ctr, 1).reshape(-1)[:n].view(st["x"].shape) < math.floor((1.0 - p) * (1 << 32))
    return tuple(t.detach().double() / (1.0 - p) * stay for t in (st["x"], st["dy"]))


def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "qk_norm_rope": _exact_norm_rope, "dropout": _exact_dropout}[case["op"]](st)
