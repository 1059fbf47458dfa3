"""Cases of the fused language-model products: 4-bit decode products, the gated feed-forward
block and the softmax cross entropy of a linear head.

``run`` computes a case in elementary torch operations, or through ``vkblas_b200`` where ``own``
is true.  All weights are N x K (one row per output), as the decode GEMV takes them.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # --- 4-bit weights, decode
        # One token through a square attention projection: the smallest call, where latency counts.
        dict(name="q4 token 4096x4096", op="q4", type="fp16", M=1, N=4096, K=4096, group=128, zeros=False),
        # One token through a down projection with zero points and finer groups.
        dict(name="q4 token 14336->4096", op="q4", type="bf16", M=1, N=4096, K=14336, group=64, zeros=True),
        # A decode batch through an odd-sized projection: K ends inside a group, N inside a tile.
        dict(name="q4 batch odd", op="q4", type="fp16", M=13, N=11003, K=4100, group=32, zeros=True),
        # --- gated feed-forward block
        # One token through the block's two projections.
        dict(name="gated token", op="gated", type="bf16", M=1, H=4096, F=14336, act="silu", save=False),
        # A small decode batch and an odd inner width.
        dict(name="gated batch odd", op="gated", type="fp16", M=9, H=2048, F=5461, act="gelu", save=False),
        # A prompt of ragged length.
        dict(name="gated prompt", op="gated", type="bf16", M=509, H=4096, F=11008, act="silu", save=False),
        # The forward pass of a training step, which keeps both projections.
        dict(name="gated train forward", op="gated", type="bf16", M=4096, H=4096, F=14336, act="silu", save=True),
        # Its backward pass.
        dict(name="gated train backward", op="gated_bwd", type="bf16", M=4096, H=4096, F=14336, act="silu"),
        # A small model's backward pass with odd token count and inner width.
        dict(name="gated backward odd", op="gated_bwd", type="fp16", M=1001, H=1024, F=2731, act="gelu_tanh"),
        # --- cross entropy of a linear head
        # Scoring a prompt: losses alone.
        dict(name="xent score", op="xent", type="bf16", T=1023, V=32000, H=4096, ignored=0.0),
        # A training step over a large vocabulary: losses and both gradients.
        dict(name="xent train", op="xent_train", type="bf16", T=4096, V=128000, H=4096, ignored=0.1),
        # A small model's step, odd token count and vocabulary.
        dict(name="xent train odd", op="xent_train", type="fp16", T=777, V=50021, H=1024, ignored=0.3),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(["q4", "q4", "gated", "gated", "gated_bwd", "xent", "xent_train"])
    t = rng.choice(["fp16", "bf16"])
    if op == "q4":
        return dict(op=op, type=t, M=rng.randint(1, 16), N=_log(rng, 500, 14336), K=_log(rng, 256, 14336, rng.choice([1, 2, 32, 128])),
                    group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
    act = rng.choice(["silu", "gelu", "gelu_tanh"])
    if op == "gated":
        return dict(op=op, type=t, M=_log(rng, 1, 4096), H=_log(rng, 256, 4096, 8), F=_log(rng, 500, 14336, rng.choice([1, 8, 128])), act=act,
                    save=rng.random() < 0.5)
    if op == "gated_bwd":
        return dict(op=op, type=t, M=_log(rng, 16, 4096), H=_log(rng, 256, 4096, 8), F=_log(rng, 500, 14336, rng.choice([1, 8, 128])), act=act)
    return dict(op=op, type=t, T=_log(rng, 16, 4096), V=_log(rng, 2000, 128000, rng.choice([1, 8, 128])), H=_log(rng, 256, 4096, 8),
                ignored=rng.choice([0.0, 0.2]))


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(t)

    s = dict(case=case)
    if case["op"] == "q4":
        M, N, K, G = case["M"], case["N"], case["K"], case["group"]
        ng = -(-K // G)
        # Two weights a byte, the even k in the low half; scales of weights with spread 1/sqrt(K).
        s["q"] = torch.randint(0, 256, (N, -(-K // 2)), device="cuda", generator=g, dtype=torch.uint8)
        s["scales"] = (torch.rand(N, ng, device="cuda", generator=g) + 0.5).mul_(0.25 / math.sqrt(K)).to(t)
        s["zeros"] = torch.randint(4, 12, (N, ng), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
        s["x"] = normal(M, K)
        if own:
            import vkblas_b200 as vk
            s["w"] = vk.q4_pack_tensors(s["q"], s["scales"], s["zeros"], K, G)
        return s
    if case["op"] in ("gated", "gated_bwd"):
        M, H, F = case["M"], case["H"], case["F"]
        s["x"] = normal(M, H)
        s["wg"] = normal(F, H, scale=1.5 / math.sqrt(H))
        s["wu"] = normal(F, H, scale=1.0 / math.sqrt(H))
        if case["op"] == "gated_bwd":
            # What the forward pass kept, and the gradient that comes from the down projection.
            s["g"] = normal(M, F, scale=1.5)
            s["u"] = normal(M, F)
            s["dh"] = normal(M, F, scale=0.05)
        return s
    T, V, H = case["T"], case["V"], case["H"]
    s["w"] = normal(V, H, scale=1.2 / math.sqrt(H))
    s["targets"] = torch.randint(0, V, (T,), device="cuda", generator=g)
    # A trained model's hidden states lean towards the row of the token that follows.
    lean = torch.rand(T, 1, device="cuda", generator=g) * 12
    x = torch.randn(T, H, device="cuda", generator=g) + s["w"][s["targets"]].float() * lean
    s["x"] = x.to(t)
    drop = torch.rand(T, device="cuda", generator=g) < case["ignored"]
    s["targets"][drop] = -100
    n = max(1, int((~drop).sum()))
    s["dloss"] = torch.full((T,), 1.0 / n, device="cuda")
    return s


# ------------------------------------------------------------------------------------ one pass
def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    a = math.sqrt(2 / math.pi)
    th = torch.tanh(a * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * a * (1 + 3 * 0.044715 * g * g)


def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(case, state)


def _run_own(case, s):
    import vkblas_b200 as vk
    op = case["op"]
    if op == "q4":
        return vk.gemv_q4_tensors(s["x"], s["w"])
    if op == "gated":
        r = vk.gated_tensors(s["x"], s["wg"], s["wu"], case["act"], save=case["save"])
        return dict(h=r[0], g=r[1], u=r[2]) if case["save"] else dict(h=r)
    if op == "gated_bwd":
        dx, dwg, dwu = vk.gated_backward_tensors(s["dh"], s["g"], s["u"], s["x"], s["wg"], s["wu"], case["act"])
        return dict(dx=dx, dwg=dwg, dwu=dwu)
    loss, lse = vk.linear_xent_tensors(s["x"], s["w"], s["targets"], ignore_index=-100)
    if op == "xent":
        return dict(loss=loss, lse=lse)
    dx, dw = vk.linear_xent_backward_tensors(s["dloss"], lse, s["x"], s["w"], s["targets"], ignore_index=-100)
    return dict(loss=loss, lse=lse, dx=dx, dw=dw)


def _run_plain(case, s):
    op, t = case["op"], TYPES[case["type"]]
    if op == "q4":
        K, G = case["K"], case["group"]
        q = torch.stack((s["q"] & 15, s["q"] >> 4), -1).flatten(1)[:, :K].float()
        z = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(G, 1)[:, :K]
        w = (q - z) * s["scales"].float().repeat_interleave(G, 1)[:, :K]
        return (s["x"].float() @ w.T).to(t)
    x = s["x"].float()
    if op == "gated":
        g, u = x @ s["wg"].float().T, x @ s["wu"].float().T
        h = (_act(g, case["act"])[0] * u).to(t)
        return dict(h=h, g=g.to(t), u=u.to(t)) if case["save"] else dict(h=h)
    if op == "gated_bwd":
        dh = s["dh"].float()
        a, da = _act(s["g"].float(), case["act"])
        dg, du = dh * s["u"].float() * da, dh * a
        dx = dg @ s["wg"].float() + du @ s["wu"].float()
        return dict(dx=dx.to(t), dwg=(dg.T @ x).to(t), dwu=(du.T @ x).to(t))
    w = s["w"].float()
    z = x @ w.T
    m = z.amax(1)
    lse = (z - m[:, None]).exp().sum(1).log() + m
    keep = s["targets"] != -100
    at = s["targets"].clamp(min=0)[:, None]
    loss = torch.where(keep, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    if op == "xent":
        return dict(loss=loss, lse=lse)
    d = (z - lse[:, None]).exp_()
    del z
    d.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
    d *= torch.where(keep, s["dloss"], torch.zeros_like(lse))[:, None]
    return dict(loss=loss, lse=lse, dx=(d @ w).to(t), dw=(d.T @ x).to(t))


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare_plain(case, seed)
    f64 = torch.float64
    op = case["op"]
    if op == "q4":
        N, K, G = case["N"], case["K"], case["group"]
        y = torch.zeros(case["M"], N, device="cuda", dtype=f64)
        x = s["x"].to(f64)
        k = torch.arange(K, device="cuda")
        for i in range(s["scales"].shape[1]):
            ks = k[i * G:(i + 1) * G]
            nib = (s["q"][:, ks // 2].to(torch.int32) >> (4 * (ks % 2)).to(torch.int32)) & 15
            z = 8 if s["zeros"] is None else s["zeros"][:, i:i + 1].to(torch.int32)
            y += (x[:, ks] @ (nib - z).to(f64).T) * s["scales"][:, i].to(f64)
        return y
    if op in ("gated", "gated_bwd"):
        x, wg, wu = (s[n].to(f64) for n in ("x", "wg", "wu"))
        if op == "gated":
            g, u = torch.einsum("mh,fh->mf", x, wg), torch.einsum("mh,fh->mf", x, wu)
        else:
            g, u = s["g"].to(f64), s["u"].to(f64)
        with torch.enable_grad():
            gl = g.detach().requires_grad_()
            a = {"silu": lambda v: v / (1 + torch.exp(-v)),
                 "gelu": lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
                 "gelu_tanh": lambda v: v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}[case["act"]](gl)
            if op == "gated_bwd":
                a.backward(s["dh"].to(f64) * u)
        a = a.detach()
        if op == "gated":
            return dict(h=a * u, g=g, u=u) if case["save"] else dict(h=a * u)
        dg, du = gl.grad, s["dh"].to(f64) * a
        return dict(dx=torch.cat((dg, du), 1) @ torch.cat((wg, wu), 0), dwg=torch.einsum("mf,mh->fh", dg, x),
                    dwu=torch.einsum("mf,mh->fh", du, x))
    x, w = s["x"].to(f64), s["w"].to(f64)
    T = case["T"]
    loss, lse = torch.zeros(T, device="cuda", dtype=f64), torch.zeros(T, device="cuda", dtype=f64)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w) if op == "xent_train" else None
    for i in range(0, T, 1024):                      # token by token alike: rows in turn
        z = x[i:i + 1024] @ w.T
        tg = s["targets"][i:i + 1024]
        rows = torch.nonzero(tg != -100)[:, 0]
        lse[i:i + 1024] = torch.logsumexp(z, 1)
        loss[i + rows] = lse[i + rows] - z[rows, tg[rows]]
        if op == "xent_train":
            p = torch.softmax(z, 1)
            p[rows, tg[rows]] -= 1
            c = torch.zeros(len(tg), device="cuda", dtype=f64)
            c[rows] = s["dloss"][i + rows].to(f64)
            p *= c[:, None]
            dx[i:i + 1024] = p @ w
            dw += p.T @ x[i:i + 1024]
    return dict(loss=loss, lse=lse, dx=dx, dw=dw) if op == "xent_train" else dict(loss=loss, lse=lse)


def prepare_plain(case, seed):
    """prepare() without the framework's laid-out weights."""
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept


def work(case):
    op = case["op"]
    if op == "q4":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"])
        return dict(bytes=N * -(-K // 2) + N * groups * (3 if case["zeros"] else 2) + 2 * M * (N + K), flops=2 * M * N * K)
    if op in ("gated", "gated_bwd"):
        M, H, F = case["M"], case["H"], case["F"]
        if op == "gated":
            return dict(bytes=2 * (M * H + 2 * F * H + M * F * (3 if case["save"] else 1)), flops=4 * M * F * H)
        return dict(bytes=2 * (3 * M * F + 2 * M * H + 4 * F * H), flops=8 * M * F * H)
    T, V, H = case["T"], case["V"], case["H"]
    if op == "xent":
        return dict(bytes=2 * (T * H + V * H) + 16 * T, flops=2 * T * V * H)
    return dict(bytes=4 * (T * H + V * H) + 20 * T, flops=6 * T * V * H)
