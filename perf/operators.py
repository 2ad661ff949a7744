"""Cases of the linear-attention and fused-linear operators: what each call has
in hand, the operators in plain torch, and the framework's own calls.

Two families, as a sequential recommender runs them together in one encoder
block (a decayed linear attention over the history, and the linear layers
around it with bias, activation and residual in one product):

``attn``   linear attention with a decay for each head, over whole histories
``train``  the same with its backward pass
``step``   one new interaction for each user, on the states kept for them
``linear`` y = act(x W^T + b) + r
``ltrain`` the same with its backward pass
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 128  # positions that the plain form treats as one block


def listed():
    return [
        # one user's next click on an idle server: latency alone
        dict(name="step_one_user", op="step", B=1, H=2, Dk=32, Dv=32, dtype="bf16", idle=0.0),
        # a serving batch of users, some of them without a new event
        dict(name="step_user_batch", op="step", B=4096, H=4, Dk=64, Dv=64, dtype="bf16", idle=0.1),
        # the same with head sizes that are no power of two
        dict(name="step_odd_heads", op="step", B=777, H=3, Dk=40, Dv=56, dtype="fp16", idle=0.0),
        # a batch of users' histories, ragged and padded on the left, into outputs and states
        dict(name="attn_histories", op="attn", B=1024, H=2, L=200, Dk=64, Dv=64, dtype="bf16", pad="left", carry=False),
        # few very long histories, continued from a kept state
        dict(name="attn_long", op="attn", B=2, H=8, L=16384, Dk=128, Dv=128, dtype="bf16", pad="none", carry=True),
        # the benchmark's training batch of short histories
        dict(name="train_short", op="train", B=8192, H=2, L=50, Dk=32, Dv=32, dtype="bf16", pad="left", carry=False),
        # training on long histories
        dict(name="train_long", op="train", B=8, H=8, L=4096, Dk=64, Dv=64, dtype="bf16", pad="right", carry=False),
        # full precision, odd sizes, with the state's gradients (a history cut into parts)
        dict(name="train_fp32_odd", op="train", B=33, H=3, L=333, Dk=48, Dv=40, dtype="fp32", pad="left", carry=True),
        # one position of a few users through a feed-forward's first product
        dict(name="linear_few_rows", op="linear", M=8, K=256, N=1024, dtype="bf16", act="gelu", bias=True, residual=False),
        # a training batch through the feed-forward's second product, with the residual
        dict(name="ltrain_narrow", op="ltrain", M=409600, K=64, N=64, dtype="bf16", act="none", bias=True, residual=True),
        # a wider encoder's feed-forward, ragged row count
        dict(name="ltrain_ffn", op="ltrain", M=25601, K=256, N=1024, dtype="bf16", act="gelu", bias=True, residual=False),
        # a large product, bound by the matrix cores
        dict(name="linear_large", op="linear", M=16384, K=4096, N=4096, dtype="bf16", act="silu", bias=True, residual=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["attn", "train", "step", "linear", "ltrain"])
    if op in ("attn", "train", "step"):
        H = rng.randint(1, 8)
        Dk = rng.choice([32, 64, 128, rng.randint(8, 128)])
        Dv = rng.choice([Dk, Dk, rng.randint(8, 128)])
        if op == "step":
            B = log(1, max(1, 2**26 // (H * Dk * Dv)))
            return dict(op=op, B=B, H=H, Dk=Dk, Dv=Dv, dtype=dtype, idle=rng.choice([0.0, 0.25]))
        L = log(1, 16384 if op == "attn" else 4096)
        B = log(1, max(1, min(8192, 2**22 // (H * L))))
        return dict(op=op, B=B, H=H, L=L, Dk=Dk, Dv=Dv, dtype=dtype,
                    pad=rng.choice(["none", "left", "right"]), carry=rng.random() < 0.5)
    N = rng.choice([64, 128, 256, 1024, log(8, 4096)])
    K = rng.choice([64, 128, 256, 1024, log(8, 4096)])
    most = 2**38 if dtype != "fp32" else 2**35
    if op == "ltrain":
        most //= 4
    M = log(1, max(1, min(409600, most // (N * K))))
    return dict(op=op, M=M, K=K, N=N, dtype=dtype, act=rng.choice(["none", "relu", "gelu", "silu"]),
                bias=rng.random() < 0.75, residual=rng.random() < 0.5)


def _head_decays(H):
    # from a horizon of some ten interactions to one of some hundreds
    x = torch.linspace(3.0, 9.0, H, dtype=torch.float64) if H > 1 else torch.tensor([5.0], dtype=torch.float64)
    return torch.log1p(-(2.0 ** -x)).float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    s = {"case": case}
    if case["op"] in ("attn", "train"):
        B, H, L, Dk, Dv = (case[n] for n in ("B", "H", "L", "Dk", "Dv"))
        # as they leave one projection: heads side by side for each position
        s["q"], s["k"], s["v"] = (normal(B, L, H, d).transpose(1, 2) for d in (Dk, Dk, Dv))
        s["log_decay"] = _head_decays(H)
        s["mask"] = None
        if case["pad"] != "none":
            length = torch.randint(1, L + 1, (B, 1), device="cuda", generator=gen)
            at = torch.arange(L, device="cuda")[None]
            s["mask"] = at < length if case["pad"] == "right" else at >= L - length
        s["state0"] = normal(B, H, Dk, Dv, dtype=torch.float32, scale=2.0) if case["carry"] else None
        if case["op"] == "train":
            s["dout"] = normal(B, L, H, Dv).transpose(1, 2)
            s["dstate"] = normal(B, H, Dk, Dv, dtype=torch.float32, scale=0.1) if case["carry"] else None
    elif case["op"] == "step":
        B, H, Dk, Dv = (case[n] for n in ("B", "H", "Dk", "Dv"))
        s["q"], s["k"], s["v"] = (normal(B, H, d) for d in (Dk, Dk, Dv))
        s["log_decay"] = _head_decays(H)
        s["active"] = None
        if case["idle"]:
            s["active"] = torch.rand(B, device="cuda", generator=gen) >= case["idle"]
        s["state"] = normal(B, H, Dk, Dv, dtype=torch.float32, scale=2.0)
    else:
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = normal(M, K)
        s["weight"] = normal(N, K, scale=1.0 / math.sqrt(K))
        s["bias"] = normal(N, scale=0.1) if case["bias"] else None
        s["residual"] = normal(M, N) if case["residual"] else None
        if case["op"] == "ltrain":
            s["dy"] = normal(M, N)
    return s


# -- the plain forms ----------------------------------------------------------


def _plain_attention(q, k, v, log_decay, mask, state0):
    """Blocks of CHUNK positions: products within each block, one state for
    each block, and the states joined by the decays between the blocks."""
    B, H, L, Dk = q.shape
    Dv = v.shape[-1]
    C = min(CHUNK, L)
    T = -(-L // C)

    def blocks(t):
        return torch.nn.functional.pad(t, (0, 0, 0, T * C - L)).reshape(B, H, T, C, t.shape[-1])

    valid = torch.ones(B, L, dtype=torch.bool, device=q.device) if mask is None else mask
    valid = torch.nn.functional.pad(valid, (0, T * C - L)).reshape(B, 1, T, C)
    q, k, v = (torch.where(valid[..., None], blocks(t), 0.0) for t in (q, k, v))
    ld = log_decay.view(1, H, 1, 1)
    count = valid.float().cumsum(-1)  # [B, 1, T, C]: valid positions up to here
    total = count[..., -1:]
    gap = (count[..., :, None] - count[..., None, :]).clamp(min=0.0)
    causal = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    weight = torch.where(causal, torch.exp(ld[..., None] * gap), 0.0)
    inside = ((q @ k.transpose(-1, -2)) * weight) @ v
    added = (k * torch.exp(ld * (total - count))[..., None]).transpose(-1, -2) @ v  # [B, H, T, Dk, Dv]
    end = total.squeeze(-1).cumsum(-1)  # [B, 1, T]
    start = end - total.squeeze(-1)
    far = (torch.cat([start, end[..., -1:]], -1)[..., :, None] - end[..., None, :]).clamp(min=0.0)
    before = torch.ones(T + 1, T, dtype=torch.bool, device=q.device).tril(-1)
    join = torch.where(before, torch.exp(ld * far), 0.0)  # [B, H, T+1, T]
    states = (join @ added.reshape(B, H, T, Dk * Dv)).reshape(B, H, T + 1, Dk, Dv)
    if state0 is not None:
        reach = torch.cat([start, end[..., -1:]], -1)[..., None, None]
        states = states + torch.exp(ld[..., None] * reach) * state0[:, :, None]
    inter = (q * torch.exp(ld * count)[..., None]) @ states[:, :, :-1]
    out = (inside + inter).reshape(B, H, T * C, Dv)[:, :, :L] / math.sqrt(Dk)
    return out, states[:, :, -1]


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_linear(x, weight, bias, residual, act):
    z = x @ weight.t()
    if bias is not None:
        z = z + bias
    y = _plain_act(z, act)
    return y if residual is None else y + residual


def _plain(s):
    case = s["case"]
    if case["op"] == "attn":
        out, state = _plain_attention(s["q"].float(), s["k"].float(), s["v"].float(), s["log_decay"], s["mask"], s["state0"])
        return out.to(s["q"].dtype), state
    if case["op"] == "train":
        leaves = [t.float().requires_grad_() for t in (s["q"], s["k"], s["v"])]
        leaves.append(s["log_decay"].clone().requires_grad_())
        if case["carry"]:
            leaves.append(s["state0"].clone().requires_grad_())
        out, state = _plain_attention(*leaves[:4], s["mask"], leaves[4] if case["carry"] else None)
        ends, seeds = ([out, state], [s["dout"].float(), s["dstate"]]) if case["carry"] else ([out], [s["dout"].float()])
        grads = torch.autograd.grad(ends, leaves, seeds)
        dt = s["q"].dtype
        outs = (out.detach().to(dt), *(g.to(dt) for g in grads[:3]), *grads[3:])
        return (*outs, state.detach()) if case["carry"] else outs
    if case["op"] == "step":
        q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
        new = torch.exp(s["log_decay"]).view(1, -1, 1, 1) * s["state"] + k[..., :, None] * v[..., None, :]
        out = (q[..., :, None] * new).sum(-2) / math.sqrt(case["Dk"])
        if s["active"] is not None:
            new = torch.where(s["active"].view(-1, 1, 1, 1), new, s["state"])
            out = torch.where(s["active"].view(-1, 1, 1), out, 0.0)
        s["state"].copy_(new)
        return out.to(s["q"].dtype), s["state"]
    names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    wide = {n: s[n].float() if s[n] is not None else None for n in ("x", "weight", "bias", "residual")}
    if case["op"] == "linear":
        return _plain_linear(**wide, act=case["act"]).to(s["x"].dtype)
    leaves = [wide[n].detach().clone().requires_grad_() if wide[n] is s[n] else wide[n].requires_grad_() for n in names]
    wide.update(zip(names, leaves))
    y = _plain_linear(**wide, act=case["act"])
    grads = torch.autograd.grad(y, leaves, s["dy"].float())
    return (y.detach().to(s["x"].dtype), *(g.to(s["x"].dtype) for g in grads))


# -- the framework's calls ----------------------------------------------------


def _own(s):
    from replay_amd.ops.fused_linear import fused_linear
    from replay_amd.ops.linear_attention import linear_attention, linear_attention_step

    case = s["case"]
    if case["op"] == "attn":
        return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], padding_mask=s["mask"],
                                initial_state=s["state0"], return_state=True)
    if case["op"] == "train":
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "log_decay")]
        if not case["carry"]:
            out = linear_attention(*leaves, padding_mask=s["mask"])
            return (out.detach(), *torch.autograd.grad(out, leaves, s["dout"]))
        leaves.append(s["state0"].detach().requires_grad_())
        out, state = linear_attention(*leaves[:4], padding_mask=s["mask"], initial_state=leaves[4], return_state=True)
        grads = torch.autograd.grad([out, state], leaves, [s["dout"], s["dstate"]])
        return (out.detach(), *grads, state.detach())
    if case["op"] == "step":
        return linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], active=s["active"]), s["state"]
    if case["op"] == "linear":
        return fused_linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
    leaves = {n: s[n].detach().requires_grad_() for n in ("x", "weight", "bias", "residual") if s[n] is not None}
    y = fused_linear(leaves["x"], leaves["weight"], leaves.get("bias"), activation=case["act"], residual=leaves.get("residual"))
    return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), s["dy"]))


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -- what a pass cannot do without --------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "step":
        rows = case["B"] * case["H"]
        return {"bytes": rows * (size * 2 * (case["Dk"] + case["Dv"]) + 8 * case["Dk"] * case["Dv"]),
                "flops": rows * 5 * case["Dk"] * case["Dv"]}
    if case["op"] in ("attn", "train"):
        B, H, L, Dk, Dv = (case[n] for n in ("B", "H", "L", "Dk", "Dv"))
        rows, states = B * H * L, 4 * B * H * Dk * Dv
        if case["op"] == "attn":
            return {"bytes": rows * size * 2 * (Dk + Dv) + states * (2 if case["carry"] else 1), "flops": rows * 4 * Dk * Dv}
        return {"bytes": rows * size * (4 * Dk + 4 * Dv) + states * (4 if case["carry"] else 0), "flops": rows * 14 * Dk * Dv}
    M, K, N = case["M"], case["K"], case["N"]
    extra = M * N if case["residual"] else 0
    if case["op"] == "linear":
        return {"bytes": size * (M * K + N * K + M * N + extra), "flops": 2 * M * N * K}
    return {"bytes": size * (2 * M * K + 2 * N * K + 2 * M * N + 2 * extra), "flops": 6 * M * N * K}


# -- from the definitions, in 64 bits -----------------------------------------


def _exact_attention(s, case):
    """Every pair of positions, a few users at a time; gradients by their formulas."""
    B, H, L, Dk, Dv = (case[n] for n in ("B", "H", "L", "Dk", "Dv"))
    ld = s["log_decay"].double().view(1, H, 1, 1)
    train = case["op"] == "train"
    parts = []
    step = max(1, int(2**28 // (H * L * L)))
    causal = torch.ones(L, L, dtype=torch.bool, device="cuda").tril()
    for lo in range(0, B, step):
        at = slice(lo, min(B, lo + step))
        valid = torch.ones(at.stop - lo, L, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][at]
        valid = valid[:, None, :, None].double()
        q, k, v = (s[n][at].double() * valid for n in ("q", "k", "v"))
        n = valid.cumsum(2)  # [b, 1, L, 1]
        gap = (n - n.transpose(2, 3)).clamp(min=0)
        decay = torch.exp(ld * gap) * causal
        from_start = torch.exp(ld * n)  # [b, H, L, 1]
        last = n[:, :, -1:]
        to_end = torch.exp(ld * (last - n))
        whole = torch.exp(ld * last)
        root = 1.0 / math.sqrt(Dk)
        qk = q @ k.transpose(2, 3)
        out = (qk * decay) @ v * root
        state = (k * to_end).transpose(2, 3) @ v
        s0 = s["state0"][at].double() if s["state0"] is not None else None
        if s0 is not None:
            out = out + (q @ s0) * from_start * root
            state = state + whole * s0
        if not train:
            parts.append((out, state))
            continue
        do = s["dout"][at].double() * valid * root
        dov = do @ v.transpose(2, 3)
        dq = (dov * decay) @ k
        dk = (dov * decay).transpose(2, 3) @ q
        dv = (qk * decay).transpose(2, 3) @ do
        dld = (gap * decay * qk * dov).sum((2, 3))
        if s0 is None:
            parts.append((out, dq, dk, dv, dld))
            continue
        ds = s["dstate"][at].double()
        dq = dq + from_start * (do @ s0.transpose(2, 3))
        dk = dk + to_end * (v @ ds.transpose(2, 3))
        dv = dv + to_end * (k @ ds)
        ds0 = (q * from_start).transpose(2, 3) @ do + whole * ds
        dld = dld + (n * from_start * (q @ s0) * do).sum((2, 3))
        dld = dld + ((last - n) * to_end * (k @ ds) * v).sum((2, 3)) + (last * whole * s0 * ds).sum((2, 3))
        # a masked position takes no part: its gradients are zero
        parts.append((out, dq * valid, dk * valid, dv * valid, dld, ds0, state))
    joined = [torch.cat(p) for p in zip(*parts)]
    if train:
        joined[4] = joined[4].sum(0)
    return tuple(joined)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("attn", "train"):
        return _exact_attention(s, case)
    if case["op"] == "step":
        q, k, v, old = (s[n].double() for n in ("q", "k", "v", "state"))
        decay = torch.exp(s["log_decay"].double())[None, :, None, None]
        new = decay * old + torch.einsum("bhi,bhj->bhij", k, v)
        out = torch.einsum("bhi,bhij->bhj", q, new) * case["Dk"] ** -0.5
        if s["active"] is not None:
            on = s["active"].double()
            new = new * on[:, None, None, None] + old * (1 - on)[:, None, None, None]
            out = out * on[:, None, None]
        return out, new
    x, w = s["x"].double(), s["weight"].double()
    z = x.mm(w.T)
    if s["bias"] is not None:
        z += s["bias"].double()
    act = case["act"]
    if act == "none":
        y, slope = z, torch.ones_like(z)
    elif act == "relu":
        slope = (z > 0).double()
        y = z * slope
    elif act == "gelu":
        cdf = torch.special.ndtr(z)
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        g = torch.sigmoid(z)
        y, slope = z * g, g + z * g * (1 - g)
    if s["residual"] is not None:
        y = y + s["residual"].double()
    if case["op"] == "linear":
        return y
    dy = s["dy"].double()
    dz = dy * slope
    grads = [dz.mm(w), dz.T.mm(x)]
    if s["bias"] is not None:
        grads.append(dz.sum(0))
    if s["residual"] is not None:
        grads.append(dy)
    return (y, *grads)
