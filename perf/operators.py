"""The matrix operators of the distillation step that need no gradient, as measured cases.

  linear_i8            y = act(x W^T + b) [+ residual] with W in 8-bit integers (one scale a channel) and x quantised
                       to 8-bit integers on the way in (one scale a token): the frozen teacher's and a compressed
                       student's projections
  layernorm_linear_i8  the same product of a LayerNorm's output, which is quantised as it is normalised; the
                       normalised rows come back in bf16 too where the residual branch needs them
  newton_schulz        the orthogonal factor of every matrix of a list, by the quintic Newton-Schulz iteration: the
                       direction that the Muon update takes

Where ``own`` is false the operators are computed in elementary torch operations in 32 bits (64 where a value next to a
rounding border decides), else by the framework's kernels.
"""

import math

import torch

own = False

LN_EPS = 1e-5
NS_STEPS = 5
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
TINY = 2.0 ** -126          # the smallest scale (a row of zeros has it)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one frame of a stream through the first feed-forward product of a Large encoder: latency
        dict(name="linear, one token", op="linear", M=1, N=4096, K=1024, x="bf16", act="gelu", residual=""),
        # one 10 s utterance, the attention's output projection of a Base encoder
        dict(name="linear, one utterance", op="linear", M=499, N=768, K=768, x="bf16", act="", residual="bf16"),
        # a pruned student's second feed-forward product: an odd number of units survives, fp32 residual stream
        dict(name="linear, pruned width", op="linear", M=1497, N=768, K=1533, x="bf16", act="", residual="fp32"),
        # 16 utterances of 10 s, the second feed-forward product of a Large encoder
        dict(name="linear, batch", op="linear", M=7984, N=1024, K=4096, x="bf16", act="", residual="fp32"),
        # one second of audio, query / key / value of a Base encoder
        dict(name="ln + linear, one second", op="ln_linear", M=49, N=2304, K=768, x="bf16", act="", keep=True),
        # a pruned student's query / key / value (7 heads survive) over three utterances of different lengths
        dict(name="ln + linear, pruned heads", op="ln_linear", M=1291, N=1344, K=768, x="bf16", act="", keep=True),
        # 16 utterances of 10 s, the first feed-forward product of a Large encoder over its fp32 stream
        dict(name="ln + linear, batch", op="ln_linear", M=7984, N=4096, K=1024, x="fp32", act="gelu", keep=False),
        # one distillation head: latency
        dict(name="newton-schulz, one head", op="ns", shapes="768x768", x="fp32"),
        # what pruning leaves of two layers, gradients in bf16
        dict(name="newton-schulz, pruned", op="ns",
             shapes="448x768*6,768x448*2,1533x768,768x1533,1201x768,768x1201,512x1536*2", x="bf16"),
        # the attention projections of a Base encoder
        dict(name="newton-schulz, attention", op="ns", shapes="768x768*48", x="fp32"),
        # the feed-forward matrices of half a Large encoder
        dict(name="newton-schulz, feed-forward", op="ns", shapes="4096x1024*12,1024x4096*12", x="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "ln_linear", "ns"])
    x = rng.choice(["bf16", "fp32"])
    if op == "ns":
        todo, left = [], 6e11
        for _ in range(rng.randint(1, 4)):
            m, n, count = _log(rng, 32, 1600), _log(rng, 32, 2600), rng.randint(1, 12)
            count = max(1, min(count, int(left / _ns_flops(m, n))))
            if _ns_flops(m, n) * count <= left:
                left -= _ns_flops(m, n) * count
                todo.append("%dx%d*%d" % (m, n, count))
        return dict(op=op, shapes=",".join(todo), x=x)
    M, N, K = _log(rng, 1, 12000), _log(rng, 64, 4200), _log(rng, 64, 4200 if op == "linear" else 1280)
    M = max(1, min(M, 7984 * 4096 * 1024 // (N * K), 7984 * 5120 // (N + K)))
    act = rng.choice(["", "gelu"])
    if op == "linear":
        return dict(op=op, M=M, N=N, K=K, x=x, act=act, residual=rng.choice(["", "bf16", "fp32"]))
    return dict(op=op, M=M, N=N, K=K, x=x, act=act, keep=rng.random() < 0.5)


def _shapes(case):
    found = []
    for s in case["shapes"].split(","):
        size, _, count = s.partition("*")
        m, n = (int(v) for v in size.split("x"))
        found += [(m, n)] * int(count or 1)
    return found


def _ns_flops(m, n):
    # a step: the Gram matrix and its square are symmetric (half of each is enough), then the product with X
    m, n = min(m, n), max(m, n)
    return NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    if case["op"] == "ns":
        e = 2 if case["x"] == "bf16" else 4
        return {"bytes": sum(m * n * (e + 2) for m, n in _shapes(case)),
                "flops": sum(_ns_flops(m, n) for m, n in _shapes(case))}
    M, N, K = case["M"], case["N"], case["K"]
    b = M * K * (2 if case["x"] == "bf16" else 4) + N * K + 8 * N
    if case["op"] == "linear":
        b += M * N * {"": 2, "bf16": 4, "fp32": 8}[case["residual"]]
    else:
        b += 8 * K + 2 * M * N + (2 * M * K if case["keep"] else 0)
    return {"bytes": b, "flops": 2 * M * N * K}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _activations(g, M, K, dtype):
    """Hidden states: unit rows with a few channels an order of magnitude above the others."""
    x = torch.randn(M, K, device="cuda", generator=g)
    c = torch.exp(0.4 * torch.randn(K, device="cuda", generator=g))
    c[torch.randint(0, K, (max(1, K // 128),), device="cuda", generator=g)] *= 8.0
    return (x * c).to(dtype)


def _gradient(g, m, n, dtype):
    """A weight gradient: a few strong directions over noise, rows of different size, small in all."""
    r = min(m, n, 24)
    u = torch.randn(m, r, device="cuda", generator=g) * torch.exp(-0.15 * torch.arange(r, device="cuda"))
    v = torch.randn(r, n, device="cuda", generator=g)
    noise = torch.randn(m, n, device="cuda", generator=g)
    rows = torch.exp(0.3 * torch.randn(m, 1, device="cuda", generator=g))
    return ((u @ v / math.sqrt(r) + noise) * rows * 1e-4).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["x"]]
    if case["op"] == "ns":
        return dict(case, mats=[_gradient(g, m, n, dt) for m, n in _shapes(case)])
    M, N, K = case["M"], case["N"], case["K"]
    s = dict(case)
    s["x"] = _activations(g, M, K, dt)
    w = torch.randn(N, K, device="cuda", generator=g) / math.sqrt(K)
    s["wq"], s["ws"] = _quantise(w)
    s["bias"] = 0.1 * torch.randn(N, device="cuda", generator=g)
    if case["op"] == "linear":
        res = case["residual"]
        s["residual"] = torch.randn(M, N, device="cuda", generator=g).to(DTYPES[res]) if res else None
    else:
        s["ln_w"] = 1.0 + 0.2 * torch.randn(K, device="cuda", generator=g)
        s["ln_b"] = 0.1 * torch.randn(K, device="cuda", generator=g)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _scale(x):
    return torch.clamp(x.float().abs().amax(1) / 127.0, min=TINY)


def _quantise(x):
    """Rows to 8-bit integers: scale = max |x| / 127 in 32 bits, q = x / scale to the nearest integer, ties to even.
    The rows of q lie 16 bytes apart or a multiple of it."""
    M, K = x.shape
    scale = _scale(x)
    q = torch.zeros(M, (K + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :K]
    q.copy_(torch.round(x.double() / scale.double()[:, None]))
    return q, scale


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))


def _product(q, scale, s):
    y = q.float() @ s["wq"].float().t() * scale[:, None] * s["ws"] + s["bias"]
    return _gelu(y) if s["act"] == "gelu" else y


def _plain_linear(s):
    y = _product(*_quantise(s["x"]), s)
    if s["residual"] is None:
        return y.bfloat16()
    return (y + s["residual"].float()).to(s["residual"].dtype)


def _normalise(x, w, b):
    x = x - x.mean(1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + LN_EPS) * w + b


def _plain_ln_linear(s):
    n = _normalise(s["x"].float(), s["ln_w"], s["ln_b"])
    y = _product(*_quantise(n), s).bfloat16()
    return [y, n.bfloat16()] if s["keep"] else [y]


def _iterate(x, steps, coeffs, eps):
    """[count, m, n] with m <= n."""
    a, b, c = coeffs
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def _same(mats):
    """The places of the matrices of each shape."""
    places = {}
    for i, t in enumerate(mats):
        places.setdefault(tuple(t.shape), []).append(i)
    return places


def _orthogonal(mats, dtype):
    out = [None] * len(mats)
    for (m, n), at in _same(mats).items():
        x = torch.stack([mats[i] for i in at]).to(dtype)
        x = _iterate(x.mT.contiguous(), NS_STEPS, NS_COEFFS, NS_EPS).mT if m > n else \
            _iterate(x, NS_STEPS, NS_COEFFS, NS_EPS)
        for i, t in zip(at, (x if dtype == torch.float64 else x.bfloat16()).unbind()):
            out[i] = t
    return out


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from dphubert_amd import kernels as K

        if s["op"] == "ns":
            return K.newton_schulz(s["mats"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
        w = K.I8Rows(s["wq"], s["ws"])
        act = K.ACT_GELU if s["act"] == "gelu" else K.ACT_NONE
        if s["op"] == "linear":
            return K.linear_i8(s["x"], w, s["bias"], act=act, residual=s["residual"])
        y, n = K.layernorm_linear_i8(s["x"], s["ln_w"], s["ln_b"], w, s["bias"], act=act, eps=LN_EPS,
                                     keep_norm=s["keep"])
        return [y, n] if s["keep"] else [y]
    if s["op"] == "ns":
        return _orthogonal(s["mats"], torch.float32)
    return _plain_linear(s) if s["op"] == "linear" else _plain_ln_linear(s)


# ---- in 64 bits --------------------------------------------------------------------------------------------------
def _exact_product(x, s):
    """x [M, K] float64: every token's scale is a 32-bit number by definition, the rest is not rounded."""
    scale = (x.abs().amax(1).float() / 127.0).clamp(min=TINY).double()
    q = torch.round(x / scale[:, None])
    y = torch.matmul(q, s["wq"].double().t()) * torch.outer(scale, s["ws"].double()) + s["bias"].double()
    return y * torch.special.ndtr(y) if s["act"] == "gelu" else y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ns":
        found = []
        for t in s["mats"]:
            x = t.double().t().contiguous() if t.shape[0] > t.shape[1] else t.double()
            x = x / (torch.linalg.matrix_norm(x) + NS_EPS)
            a, b, c = NS_COEFFS
            for _ in range(NS_STEPS):
                gram = torch.mm(x, x.t())
                x = torch.mm(torch.addmm(gram, gram, gram, beta=b, alpha=c), x).add_(x, alpha=a)
            found.append(x.t().contiguous() if t.shape[0] > t.shape[1] else x)
        return found
    x = s["x"].double()
    if case["op"] == "linear":
        y = _exact_product(x, s)
        return y if s["residual"] is None else y + s["residual"].double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).pow(2).mean(1, keepdim=True)
    n = (x - mean) / torch.sqrt(var + LN_EPS) * s["ln_w"].double() + s["ln_b"].double()
    y = _exact_product(n, s)
    return [y, n] if case["keep"] else [y]
