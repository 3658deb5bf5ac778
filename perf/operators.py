"""The products of a gated feed-forward layer: what they compute in plain torch operations, and the
library's calls for the same.

A case names one operator ("op") and its sizes.  M counts tokens (rows of the activations); K is the depth of the
products, N the number of channels; "pad" is how many elements lie between the end of a row of an input and the
next row.

  quant     rows to 8-bit integers with one scale each         Q, s
  i8gemm    8-bit product, a scale for each token and channel   C
  gated     act(X Wg^T) o (X Wu^T)                              H, with "save" also G and U
  i8gated   the same on 8-bit operands                          H
  grad      its gradients                                       dX, dWg, dWu
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GATES = ("silu", "gelu", "gelu_tanh")


def _case(name, op, type_, M, N, K, pad=0, gate="silu", save=False):
    return {"name": name, "op": op, "type": type_, "M": M, "N": N, "K": K, "pad": pad, "gate": gate, "save": save}


def listed():
    return [
        # one decoding step of a small batch: launch latency
        _case("quant 8 tokens", "quant", "bf16", 8, 1, 4096),
        # a long prompt's activations: bandwidth
        _case("quant prompt", "quant", "bf16", 16384, 1, 8192),
        # one token through an output projection: the weights' bytes
        _case("i8 token", "i8gemm", "bf16", 1, 4096, 4096),
        # sizes and strides that fit no tile, results kept in 32 bits
        _case("i8 ragged", "i8gemm", "f32", 1000, 5003, 2501, pad=7),
        # a prompt: the matrix cores
        _case("i8 prompt", "i8gemm", "bf16", 8192, 8192, 8192),
        # one token through both projections
        _case("gated token", "gated", "bf16", 1, 12288, 4096),
        # a training step's forward pass, with what its backward pass reads
        _case("gated train", "gated", "bf16", 8192, 12288, 4096, save=True),
        # a short ragged prompt, the other 16-bit type, another gate
        _case("gated ragged", "gated", "f16", 333, 2751, 1030, pad=2, gate="gelu_tanh"),
        # a decoding batch on 8-bit weights
        _case("i8 gated batch", "i8gated", "bf16", 16, 12288, 4096),
        # a short prompt on 8-bit weights
        _case("i8 gated prompt", "i8gated", "f16", 2048, 12288, 4096, gate="gelu_tanh"),
        # a training step's backward pass
        _case("grad train", "grad", "bf16", 8192, 12288, 4096),
        # a small layer with ragged sizes
        _case("grad ragged", "grad", "f16", 509, 1367, 770, pad=6, gate="gelu"),
    ]


def draw(rng):
    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        unit = rng.choice((1, 1, 8, 64))
        return max(lo, n // unit * unit)

    op = rng.choice(("quant", "i8gemm", "gated", "i8gated", "grad"))
    while True:
        M, N, K = size(1, 16384 if op == "quant" else 8192), size(64, 12288), size(64, 8192)
        if op == "quant" or M * N * K <= 8192 * 12288 * 4096:
            break
    type_ = rng.choice(("f32", "f16", "bf16") if op in ("quant", "i8gemm", "i8gated") else ("f16", "bf16"))
    return {"op": op, "type": type_, "M": M, "N": 1 if op == "quant" else N, "K": K,
            "pad": rng.choice((0, 0, 0, rng.randrange(1, 65))), "gate": rng.choice(GATES),
            "save": op == "gated" and rng.random() < 0.5}


def work(case):
    M, N, K = case["M"], case["N"], case["K"]
    e = TYPES[case["type"]].itemsize
    op = case["op"]
    if op == "quant":
        return {"bytes": M * K * (e + 1) + 4 * M, "flops": 3 * M * K}
    if op == "i8gemm":
        return {"bytes": M * K + N * K + 4 * (M + N) + e * M * N, "flops": 2 * M * N * K}
    if op == "gated":
        return {"bytes": e * (M * K + 2 * N * K + (3 if case["save"] else 1) * M * N), "flops": 4 * M * N * K}
    if op == "i8gated":
        return {"bytes": M * K + 2 * N * K + 4 * (M + 2 * N) + e * M * N, "flops": 4 * M * N * K}
    return {"bytes": e * (3 * M * N + 2 * M * K + 4 * N * K), "flops": 8 * M * N * K}


class _Maker:
    """Random matrices on the GPU whose rows lie `pad` elements apart."""

    def __init__(self, seed, pad):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.pad = pad

    def normal(self, rows, cols, std, dtype):
        x = torch.randn(rows, cols + self.pad, generator=self.gen, device="cuda", dtype=torch.float32)
        return x.mul_(std).to(dtype)[:, :cols]

    def whole(self, rows, cols):
        x = torch.randn(rows, cols + self.pad, generator=self.gen, device="cuda", dtype=torch.float32)
        return x.mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)[:, :cols]

    def scales(self, n, around):
        return torch.rand(n, generator=self.gen, device="cuda", dtype=torch.float32).add_(0.5).mul_(around)


def prepare(case, seed):
    op, M, N, K = case["op"], case["M"], case["N"], case["K"]
    dtype = TYPES[case["type"]]
    make = _Maker(seed, case["pad"])

    def out(rows, cols, t=dtype):
        return torch.empty(rows, cols, device="cuda", dtype=t)

    st = {"case": case}
    if op == "quant":
        # activations with a few channels that stand out, as a layer's input has them
        x = make.normal(M, K, 1.0, torch.float32)
        channels = torch.randint(0, K, (max(1, K // 512),), generator=make.gen, device="cuda")
        x[:, channels] *= 12.0
        st["X"] = x._base.to(dtype)[:, :K] if x._base is not None else x.to(dtype)
        st["Q"], st["s"] = out(M, K, torch.int8), out(1, M, torch.float32)[0]
    elif op == "i8gemm":
        st["A"], st["sA"] = make.whole(M, K), make.scales(M, 0.02)
        st["B"], st["sB"] = make.whole(N, K), make.scales(N, 0.02 / math.sqrt(K))
        st["C"] = out(M, N)
    elif op == "i8gated":
        st["X"], st["sX"] = make.whole(M, K), make.scales(M, 0.025)
        st["Wg"], st["sg"] = make.whole(N, K), make.scales(N, 0.025 / math.sqrt(K))
        st["Wu"], st["su"] = make.whole(N, K), make.scales(N, 0.025 / math.sqrt(K))
        st["H"] = out(M, N)
    else:
        st["X"] = make.normal(M, K, 1.0, dtype)
        st["Wg"] = make.normal(N, K, 1.0 / math.sqrt(K), dtype)
        st["Wu"] = make.normal(N, K, 1.0 / math.sqrt(K), dtype)
        if op == "gated":
            st["H"] = out(M, N)
            if case["save"]:
                st["G"], st["U"] = out(M, N), out(M, N)
        else:
            st["G"], st["U"] = make.normal(M, N, 1.0, dtype), make.normal(M, N, 1.0, dtype)
            st["dH"] = make.normal(M, N, 1.0, dtype)
            st["dX"], st["dWg"], st["dWu"] = out(M, K), out(N, K), out(N, K)
    return st


def _act(gate, g):
    if gate == "silu":
        return g / (1.0 + torch.exp(-g))
    if gate == "gelu":
        return g * 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _act_slope(gate, g):
    if gate == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    if gate == "gelu":
        return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _plain(st):
    case = st["case"]
    op, gate, dtype = case["op"], case["gate"], TYPES[case["type"]]
    if op == "quant":
        # 64 bits: quotients next to a half decide the integer
        x = st["X"].double()
        a = x.abs().amax(dim=1, keepdim=True)
        q = torch.where(a > 0, torch.round(127.0 * x / a), torch.zeros_like(x))
        return q.to(torch.int8), a[:, 0].float() / 127.0
    if op == "i8gemm":
        # 64 bits: sums of 8-bit products pass 2^24
        acc = torch.matmul(st["A"].double(), st["B"].double().t()).float()
        return (acc * st["sA"][:, None] * st["sB"][None, :]).to(dtype)
    if op == "i8gated":
        x = st["X"].double()
        g = torch.matmul(x, st["Wg"].double().t()).float() * st["sX"][:, None] * st["sg"][None, :]
        u = torch.matmul(x, st["Wu"].double().t()).float() * st["sX"][:, None] * st["su"][None, :]
        return (_act(gate, g) * u).to(dtype)
    x, wg, wu = st["X"].float(), st["Wg"].float(), st["Wu"].float()
    if op == "gated":
        g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
        h = (_act(gate, g) * u).to(dtype)
        return (h, g.to(dtype), u.to(dtype)) if case["save"] else h
    g, u, dh = st["G"].float(), st["U"].float(), st["dH"].float()
    du = dh * _act(gate, g)
    dg = dh * u * _act_slope(gate, g)
    dx = torch.matmul(dg, wg) + torch.matmul(du, wu)
    return dx.to(dtype), torch.matmul(dg.t(), x).to(dtype), torch.matmul(du.t(), x).to(dtype)


def _check(status):
    if status != 0:
        raise RuntimeError("the library returned %d" % status)


def _calls(st):
    import clblas_amd as cb
    case = st["case"]
    op, M, N, K = case["op"], case["M"], case["N"], case["K"]
    type_ = {"f32": cb.Type.F32, "f16": cb.Type.F16, "bf16": cb.Type.BF16}[case["type"]]
    gate = {"silu": cb.Gate.Silu, "gelu": cb.Gate.Gelu, "gelu_tanh": cb.Gate.GeluTanh}[case["gate"]]

    def mat(name):
        x = st.get(name)
        return (None, 0, 0) if x is None else (x, 0, x.stride(0))

    if op == "quant":
        _check(cb.quantize_rows(type_, M, K, *mat("X"), *mat("Q"), st["s"]))
        return st["Q"], st["s"]
    if op == "i8gemm":
        _check(cb.i8gemm(type_, M, N, K, *mat("A"), st["sA"], *mat("B"), st["sB"], *mat("C")))
        return st["C"]
    if op == "i8gated":
        _check(cb.gated_i8(type_, gate, M, N, K, *mat("X"), st["sX"], *mat("Wg"), st["sg"], *mat("Wu"), st["su"], *mat("H")))
        return st["H"]
    if op == "gated":
        _check(cb.gated(type_, gate, M, N, K, *mat("X"), *mat("Wg"), *mat("Wu"), *mat("H"), *mat("G"), *mat("U")))
        return (st["H"], st["G"], st["U"]) if case["save"] else st["H"]
    _check(cb.gated_grad(type_, gate, M, N, K, *mat("dH"), *mat("X"), *mat("Wg"), *mat("Wu"), *mat("G"), *mat("U"),
                         *mat("dX"), *mat("dWg"), *mat("dWu")))
    return st["dX"], st["dWg"], st["dWu"]


def run(state):
    return _calls(state) if own else _plain(state)


def exact(case, seed):
    """The definitions, element by element in 64 bits, on the inputs of `prepare`."""
    st = prepare(case, seed)
    f = {k: v.to(torch.float64) for k, v in st.items() if k in ("X", "A", "B", "Wg", "Wu", "G", "U", "dH", "sA", "sB", "sX", "sg", "su")}
    op = case["op"]
    half = torch.tensor(0.5, dtype=torch.float64, device="cuda")

    def cdf(g):  # of the standard normal distribution
        return half * torch.special.erfc(-g / math.sqrt(2.0))

    def inner(g):
        return 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)

    def act(g):
        if case["gate"] == "silu":
            return g * torch.sigmoid(g)
        return g * (cdf(g) if case["gate"] == "gelu" else torch.sigmoid(inner(g)))

    def slope(g):
        if case["gate"] == "gelu":
            return cdf(g) + g * torch.exp(-g * g / 2.0) / math.sqrt(2.0 * math.pi)
        z, dz = (g, 1.0) if case["gate"] == "silu" else (inner(g), 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * g ** 2))
        s = torch.sigmoid(z)
        return s + g * s * torch.sigmoid(-z) * dz

    if op == "quant":
        # the integer nearest to 127 x / a, by comparing 254 |x| with odd multiples of a
        x, big = f["X"].abs(), f["X"].abs().max(dim=1, keepdim=True).values
        n = torch.floor(127.0 * x / big.clamp(min=1e-300))
        over = 254.0 * x - (2.0 * n + 1.0) * big
        n = n + ((over > 0) | ((over == 0) & (n % 2 == 1))).double()
        return (torch.where(f["X"] < 0, -n, n) * (big > 0)).to(torch.int8), (big / 127.0)[:, 0]
    if op == "i8gemm":
        return (f["A"] * f["sA"][:, None]) @ (f["B"] * f["sB"][:, None]).T
    if op == "i8gated":
        x = f["X"] * f["sX"][:, None]
        return act(x @ (f["Wg"] * f["sg"][:, None]).T) * (x @ (f["Wu"] * f["su"][:, None]).T)
    if op == "gated":
        g, u = f["X"] @ f["Wg"].T, f["X"] @ f["Wu"].T
        return (act(g) * u, g, u) if case["save"] else act(g) * u
    du, dg = f["dH"] * act(f["G"]), f["dH"] * f["U"] * slope(f["G"])
    return dg @ f["Wg"] + du @ f["Wu"], dg.T @ f["X"], du.T @ f["X"]
