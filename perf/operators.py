"""Cases that measure the operators of packed language-model training: attention over packed sequences with grouped heads
(``nn_ops.attention_packed``) and the cross-entropy of a linear head that keeps no logits (``nn_ops.linear_cross_entropy``).

``run`` computes them in plain torch operations in fp32 while ``own`` is false, and through the framework's entry points while it is true.
A case is a dict of plain values; ``prepare`` builds from it, on the GPU, what a training program has in hand before the call.
"""
import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # four prompts of a few tokens through the tiny decoder's heads: launch latency is everything
        {"name": "attn_tiny_fwd", "kind": "attn", "tokens": 41, "seqs": 4, "spread": 2.0, "pad": 0, "heads": 4, "kv_heads": 4, "hd": 32, "causal": True,
         "dtype": "bf16", "train": False},
        # a fine-tuning batch of short replies, most of them shorter than a tile, grouped heads, padded rows behind the last one
        {"name": "attn_short_train", "kind": "attn", "tokens": 2500, "seqs": 96, "spread": 4.0, "pad": 60, "heads": 8, "kv_heads": 2, "hd": 64, "causal": True,
         "dtype": "fp16", "train": True},
        # the forward pass over a ragged batch of prompts (evaluation), four query heads to a key head
        {"name": "attn_prompts_fwd", "kind": "attn", "tokens": 8191, "seqs": 7, "spread": 5.0, "pad": 0, "heads": 16, "kv_heads": 4, "hd": 128, "causal": True,
         "dtype": "bf16", "train": False},
        # one micro-batch of the 1.3 B decoder (four rows of 2,048 tokens, sixteen heads of 128) with its documents packed
        {"name": "attn_llama_train", "kind": "attn", "tokens": 8192, "seqs": 14, "spread": 5.0, "pad": 0, "heads": 16, "kv_heads": 16, "hd": 128,
         "causal": True, "dtype": "bf16", "train": True},
        # one long document and a shorter one: long-context training with eight query heads to a key head
        {"name": "attn_long_train", "kind": "attn", "tokens": 16384, "seqs": 2, "spread": 6.0, "pad": 0, "heads": 16, "kv_heads": 2, "hd": 128,
         "causal": True, "dtype": "bf16", "train": True},
        # bidirectional attention of a small fp32 model, a head size that is no power of two
        {"name": "attn_fp32_train", "kind": "attn", "tokens": 1023, "seqs": 5, "spread": 2.0, "pad": 3, "heads": 4, "kv_heads": 4, "hd": 80, "causal": False,
         "dtype": "fp32", "train": True},
        # the tiny decoder's head: launch latency
        {"name": "loss_tiny_train", "kind": "loss", "rows": 200, "vocab": 256, "d": 128, "ignored": 8, "dtype": "bf16", "train": True},
        # validation loss of the 1.3 B decoder
        {"name": "loss_llama_eval", "kind": "loss", "rows": 4095, "vocab": 32000, "d": 2048, "ignored": 5, "dtype": "bf16", "train": False},
        # one micro-batch of the 1.3 B decoder: four rows of 2,047 positions that have a next token
        {"name": "loss_llama_train", "kind": "loss", "rows": 8188, "vocab": 32000, "d": 2048, "ignored": 0, "dtype": "bf16", "train": True},
        # fine-tuning in fp16: an odd vocabulary, a width that is no multiple of a tile, half of the positions are prompt and not counted
        {"name": "loss_odd_train", "kind": "loss", "rows": 1537, "vocab": 50021, "d": 1000, "ignored": 768, "dtype": "fp16", "train": True},
        # a handful of positions: the head's weights are read and their gradient is written, little is computed
        {"name": "loss_few_train", "kind": "loss", "rows": 13, "vocab": 32000, "d": 2048, "ignored": 0, "dtype": "bf16", "train": True},
        # a small model trained in fp32
        {"name": "loss_fp32_train", "kind": "loss", "rows": 777, "vocab": 5003, "d": 512, "ignored": 7, "dtype": "fp32", "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    dtype, train = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"]), rng.random() < 0.7
    if rng.random() < 0.5:
        kv, group = rng.choice([(1, 1), (4, 1), (12, 1), (16, 1), (4, 2), (2, 4), (4, 4), (1, 8), (2, 8), (2, 3), (1, 7)])
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 40])
        top = 2048 if dtype == "fp32" else 16384 * 16 // max(16, kv * group)
        tokens = _log_int(rng, 1, top)
        seqs = _log_int(rng, 1, max(1, min(tokens, 400)))
        pad = rng.choice([0, 0, rng.randint(0, tokens // 8)])
        return {"kind": "attn", "tokens": tokens, "seqs": seqs, "spread": round(6.0 * rng.random(), 2), "pad": pad,
                "heads": kv * group, "kv_heads": kv, "hd": hd, "causal": rng.random() < 0.8, "dtype": dtype, "train": train}
    small = dtype == "fp32"
    vocab, d = _log_int(rng, 200, 8000 if small else 60000), 8 * _log_int(rng, 8, 64 if small else 256)
    rows = _log_int(rng, 1, max(1, min(1024 if small else 8192, int(5e11 / vocab / d))))
    return {"kind": "loss", "rows": rows, "vocab": vocab, "d": d, "ignored": rng.choice([0, 0, rng.randint(0, rows // 2)]), "dtype": dtype, "train": train}


def _lengths(c):
    """Lengths of the packed sequences, spread over their logarithm by a factor of up to e^spread (short ones come out empty at times).  They
    belong to the case, not to the seed: another seed means other values in the same layout, as the next layer of a model has them."""
    weights = np.exp(c["spread"] * np.random.RandomState(c["tokens"] % 1009 * 401 + c["seqs"]).rand(c["seqs"]))
    cuts = np.rint(np.cumsum(weights) / weights.sum() * (c["tokens"] - c["pad"])).astype(np.int64)
    return np.diff(cuts, prepend=0).tolist()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    dt = DT[c["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)
    if c["kind"] == "attn":
        lens = _lengths(c)
        cu = np.cumsum([0] + lens).tolist()
        T, H, K, hd = c["tokens"], c["heads"], c["kv_heads"], c["hd"]
        s = {"q": randn(T, H, hd), "k": randn(T, K, hd), "v": randn(T, K, hd), "cu": torch.tensor(cu, dtype=torch.int32, device=DEV)}
        if c["train"]:
            s["do"] = randn(T, H, hd)
            for t in (s["q"], s["k"], s["v"]):
                t.requires_grad_(True)
    else:
        N, V, D = c["rows"], c["vocab"], c["d"]
        t = torch.randint(0, V, (N,), generator=g, device=DEV)
        w = torch.randn(V, D, generator=g, device=DEV) * (1.5 / D ** 0.5)
        x = torch.randn(N, D, generator=g, device=DEV) + 2.0 * w[t]      # a model that has learned something: targets stand out
        t[torch.randperm(N, generator=g, device=DEV)[: c["ignored"]]] = -100
        s = {"x": x.to(dt), "w": w.to(dt), "t": t}
        if c["train"]:
            s["gout"] = torch.tensor(8192.0 if c["dtype"] == "fp16" else 1.0, device=DEV)       # the loss scale of fp16 training
            s["x"].requires_grad_(True), s["w"].requires_grad_(True)
    s["c"] = c
    return s


def _attn_plain(q, k, v, cu, causal, do):
    """Scores of all pairs of rows, masked by sequence and order.  Rows of no sequence give zeros."""
    T, H, hd = q.shape
    G = H // k.shape[1]
    qf, kf, vf = (t.float().transpose(0, 1) for t in (q, k, v))
    kf, vf = kf.repeat_interleave(G, 0), vf.repeat_interleave(G, 0)
    scale = hd ** -0.5
    row = torch.arange(T, device=q.device)
    seq = torch.searchsorted(cu.long(), row, right=True)                # 0 before the first, len(cu) behind the last sequence
    live = (seq > 0) & (seq < cu.numel())
    mask = (seq[:, None] == seq[None, :]) & live[:, None]
    if causal:
        mask &= row[None, :] <= row[:, None]
    p = torch.matmul(qf, kf.transpose(1, 2)).mul_(scale).masked_fill_(~mask, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(~live[None, :, None], 0.0)).exp_()
    p.div_(p.sum(-1, keepdim=True).masked_fill_(~live[None, :, None], 1.0))
    out = torch.matmul(p, vf).transpose(0, 1)
    if do is None:
        return out.to(q.dtype)
    dof = do.float().transpose(0, 1)
    dv = torch.matmul(p.transpose(1, 2), dof)
    ds = torch.matmul(dof, vf.transpose(1, 2))
    delta = (dof * out.transpose(0, 1)).sum(-1, keepdim=True)           # sum_j p_ij dp_ij
    ds.sub_(delta).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(1, 2), qf)
    dk, dv = (t.view(H // G, G, T, hd).sum(1) for t in (dk, dv))
    return [t.to(q.dtype).contiguous() for t in (out, dq.transpose(0, 1), dk.transpose(0, 1), dv.transpose(0, 1))]


def _loss_plain(x, w, t, gout):
    xf, wf = x.float(), w.float()
    z = torch.matmul(xf, wf.t())
    counted = (t >= 0) & (t < w.shape[0])
    n = counted.sum().clamp(min=1)
    at = t.clamp(0, w.shape[0] - 1)[:, None]
    zt = z.gather(1, at)
    top = z.amax(1, keepdim=True)
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    loss = ((top + total.log() - zt)[:, 0] * counted).sum() / n
    if gout is None:
        return loss
    z.div_(total)
    z.scatter_add_(1, at, torch.full_like(zt, -1.0))
    z.mul_((counted * (gout / n))[:, None])
    return [loss, torch.matmul(z, wf).to(x.dtype), torch.matmul(z.t(), xf).to(w.dtype)]


def run(state):
    s, c = state, state["c"]
    if c["kind"] == "attn":
        if not own:
            with torch.no_grad():
                return _attn_plain(s["q"], s["k"], s["v"], s["cu"], c["causal"], s.get("do"))
        from supergrok15_b200.ops import nn_ops
        out = nn_ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"])
        if not c["train"]:
            return out
        return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])]
    if not own:
        with torch.no_grad():
            return _loss_plain(s["x"], s["w"], s["t"], s.get("gout"))
    from supergrok15_b200.ops import nn_ops
    loss = nn_ops.linear_cross_entropy(s["x"], s["w"], s["t"])
    if not c["train"]:
        return loss
    return [loss, *torch.autograd.grad(loss, (s["x"], s["w"]), s["gout"])]


def work(case):
    c = case
    es = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "attn":
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in _lengths(c))
        rows_q, rows_k = c["tokens"] * c["heads"] * c["hd"] * es, c["tokens"] * c["kv_heads"] * c["hd"] * es
        # forward: q, k, v in, out; with gradients: dout in, dq, dk, dv out as well (what else a backward pass reads again need not leave the chip)
        return {"bytes": (4 * rows_q + 4 * rows_k) if c["train"] else (2 * rows_q + 2 * rows_k),
                "flops": (14 if c["train"] else 4) * pairs * c["heads"] * c["hd"]}
    n, io = c["rows"] - c["ignored"], (c["vocab"] + c["rows"]) * c["d"] * es
    return {"bytes": 2 * io + 8 * c["rows"] if c["train"] else io + 8 * c["rows"], "flops": (6 if c["train"] else 2) * n * c["vocab"] * c["d"]}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    with torch.no_grad():
        if c["kind"] == "attn":
            q, k, v = (s[n].detach().double() for n in "qkv")
            do = s["do"].double() if c["train"] else None
            res = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
            G = c["heads"] // c["kv_heads"]
            for a, b in zip(s["cu"].tolist()[:-1], s["cu"].tolist()[1:]):
                if a == b:
                    continue
                for h in range(c["heads"]):
                    z = q[a:b, h] @ k[a:b, h // G].t() / c["hd"] ** 0.5
                    if c["causal"]:
                        z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(1), float("-inf"))
                    p = torch.softmax(z, 1)
                    del z
                    res[0][a:b, h] = p @ v[a:b, h // G]
                    if do is None:
                        continue
                    dp = do[a:b, h] @ v[a:b, h // G].t()
                    ds = p * (dp - (p * dp).sum(1, keepdim=True)) / c["hd"] ** 0.5
                    res[1][a:b, h] = ds @ k[a:b, h // G]
                    res[2][a:b, h // G] += ds.t() @ q[a:b, h]
                    res[3][a:b, h // G] += p.t() @ do[a:b, h]
            return res if c["train"] else res[0]
        x, w, t = s["x"].detach().double(), s["w"].detach().double(), s["t"]
        keep = t != -100
        x, t = x[keep], t[keep]
        n = max(1, int(keep.sum()))
        z = x @ w.t()
        loss = (torch.logsumexp(z, 1) - z[torch.arange(len(t), device=z.device), t]).sum() / n
        if not c["train"]:
            return loss
        p = torch.softmax(z, 1)
        p[torch.arange(len(t), device=z.device), t] -= 1.0
        p *= float(s["gout"]) / n
        dx = torch.zeros(c["rows"], c["d"], dtype=torch.float64, device=z.device)
        dx[keep] = p @ w
        return [loss, dx, p.t() @ x]
