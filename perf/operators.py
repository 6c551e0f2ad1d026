"""What is measured of the training-step operators: group normalisation with its activation (forward, and forward + backward),
the global gradient norm over a network's tensors, clipping by it, and the Adam step that takes the clip with it.

Plain forms are elementary torch operations; sums over an image or over all gradients, and the side of zero on which a ReLU's
argument lies, are computed in 64 bits there, because 32 lose them (a ReLU's gradient jumps at zero: one argument in some
millions is within a 32-bit rounding of it)."""
import math

import torch

own = False

ACTS = ("none", "relu", "leaky_relu", "silu")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS, CLIP_EPS = 1e-5, 1e-6
LR, BETA1, BETA2, ADAM_EPS = 1e-4, 0.5, 0.9, 1e-8       # the training commands' learning rate and betas


# ---- cases ------------------------------------------------------------------------------------------------------
def _gn(op, n, c, g, d, h, w, dtype, layout, act, **name):
    return {**name, "op": op, "n": n, "c": c, "groups": g, "d": d, "h": h, "w": w, "dtype": dtype, "layout": layout, "act": act}


def _nets(op, net, nf, dtype="fp32", **more):
    return {**more, "op": op, "net": net, "nf": nf, "dtype": dtype}


def listed():
    return [
        # the voxel refiner's first encoder stage (20 channels at 64^3), a batch of four, channels last
        _gn("gn", 4, 20, 4, 64, 64, 64, "fp32", "last", "leaky_relu", name="gn refiner 64^3 x4 last"),
        # the voxel decoder's widest map (32 channels at 64^3), a batch of eight in bf16, in the networks' default layout
        _gn("gn", 8, 32, 8, 64, 64, 64, "bf16", "first", "relu", name="gn decoder 64^3 x8 bf16"),
        # one image in the refiner's fourth stage: a prediction, where latency counts
        _gn("gn", 1, 160, 8, 8, 8, 8, "fp32", "last", "leaky_relu", name="gn one image 8^3"),
        # the same stages in training: forward, then the gradients of the map, the weight and the bias
        _gn("gn_train", 4, 20, 4, 64, 64, 64, "fp32", "last", "leaky_relu", name="gn train refiner 64^3 x4"),
        _gn("gn_train", 8, 32, 8, 64, 64, 64, "bf16", "first", "relu", name="gn train decoder 64^3 x8"),
        # odd sizes, a map of two dimensions, the smooth activation
        _gn("gn_train", 3, 45, 5, 1, 61, 47, "fp16", "last", "silu", name="gn train odd map fp16"),
        # gradients of the voxel refiner (48 tensors, 53 million values): what a training log reads
        _nets("norm", "refiner", 20, norm="2", name="norm refiner"),
        # the largest gradient of the generator (16 tensors), held in bf16
        _nets("norm", "generator", 64, "bf16", norm="inf", name="max norm generator bf16"),
        # clipping in place: the critic's 6 tensors, and the joint model's some 440 tensors of 100 million values
        _nets("clip", "critic", 64, norm="2", max_norm=1.0, name="clip critic"),
        _nets("clip", "joint", 20, norm="2", max_norm=1.0, name="clip joint model"),
        # the optimiser's step with the clip folded in, on the same two
        _nets("adam", "critic", 64, norm="2", max_norm=1.0, decay=0.0, step=7, name="adam critic"),
        _nets("adam", "joint", 20, norm="2", max_norm=1.0, decay=0.0, step=1000, name="adam joint model"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gn", "gn_train", "norm", "clip", "adam"))
    if op.startswith("gn"):
        groups = rng.choice((1, 2, 4, 5, 8, 16, 32))
        c = groups * _log(rng, 1, max(1, 640 // groups))
        d = rng.choice((1, _log(rng, 1, 64)))
        n, h, w = _log(rng, 1, 8), _log(rng, 1, 256 if d == 1 else 64), _log(rng, 1, 256 if d == 1 else 64)
        while n * c * d * h * w > 8 * 32 * 64 ** 3:                       # no more than the largest listed one
            n, d, h = max(1, n // 2), max(1, d // 2), max(1, h // 2)
        if c // groups * d * h * w < 4:                                   # a statistic over less than that says nothing
            h, w = h + 3, w + 5
        return _gn(op, n, c, groups, d, h, w, rng.choice(sorted(DTYPES)), rng.choice(("last", "first")), rng.choice(ACTS))
    net = rng.choice(("refiner", "critic", "generator", "joint"))
    nf = rng.randint(3, 20) if net in ("refiner", "joint") else rng.randint(5, 64)
    case = _nets(op, net, nf, rng.choice(sorted(DTYPES)), norm="2" if op == "adam" else rng.choice(("2", "2", "inf")))
    if op != "norm":
        case["max_norm"] = rng.choice((0.1, 1.0, 10.0))
    if op == "adam":
        case.update(decay=rng.choice((0.0, 0.01)), step=_log(rng, 1, 10000))
    return case


# ---- the tensors of the networks that are trained ---------------------------------------------------------------
def _refiner(nf):
    w = [2] + [nf << i for i in range(6)]
    out = []
    for i, k in enumerate((8, 4, 4, 4, 4, 4)):
        out += [(w[i + 1], w[i], k, k, k)] + [(w[i + 1],)] * 3
    out += [(w[6], w[6]), (w[6],)]
    for i, k in enumerate((4, 4, 4, 4, 8)):
        out += [(2 * w[6 - i], w[5 - i], k, k, k)] + [(w[5 - i],)] * 3
    return out + [(2 * nf, 1, 4, 4, 4), (1,)]


def _critic(nf):
    w = [1, nf, nf, 2 * nf, 4 * nf, 8 * nf]
    return [(b, a, 4, 4, 4) for a, b in zip(w[:-1], w[1:])] + [(1, 8 * nf, 4, 4, 4)]


def _generator(nf):
    w = [200, 8 * nf, 4 * nf, 2 * nf, nf, nf]
    return [s for a, b in zip(w[:-1], w[1:]) for s in ((a, b, 4, 4, 4), (b,), (b,))] + [(nf, 1, 4, 4, 4)]


def _residual(widths, c):
    out = []
    for w in widths:                                                      # two residual blocks a stage, each conv with a norm
        out += [(w, c, 3, 3), (w,), (w,), (w, w, 3, 3), (w,), (w,), (w, c, 1, 1), (w,), (w,)]
        out += [(w, w, 3, 3), (w,), (w,), (w, w, 3, 3), (w,), (w,)]
        c = w
    return out


def _joint(nf):                     # two image networks on residual encoders, with three decoders and one, and the refiner
    f = max(4, 64 * nf // 20)
    encoder = [(f, 3, 7, 7), (f,), (f,)] + _residual((f, 2 * f, 4 * f, 8 * f), f)
    decoder = _residual((4 * f, 2 * f, f, f), 8 * f) + [(f, f, 3, 3), (f,), (f,), (f,), (f, 1, 7, 7)]
    return encoder + 3 * decoder + encoder + decoder + _refiner(nf)


_NETS = {"refiner": _refiner, "critic": _critic, "generator": _generator, "joint": _joint}


def _views(flat, shapes):
    at, out = 0, []
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"].startswith("gn"):
        n, c = case["n"], case["c"]
        space = [s for s in (case["d"], case["h"], case["w"])][0 if case["d"] > 1 else 1:]
        one = [1, c] + [1] * len(space)
        fmt = {("last", 2): torch.channels_last, ("last", 3): torch.channels_last_3d}.get((case["layout"], len(space)), torch.contiguous_format)
        # a convolution's output: channels with levels and spreads of their own
        x = normal(n, c, *space) * (0.3 + normal(*one).abs()) + 0.5 * normal(*one)
        x = x.to(dtype).contiguous(memory_format=fmt)
        state = {"case": case, "x": x, "weight": 1 + 0.1 * normal(c), "bias": 0.1 * normal(c)}
        if case["op"] == "gn_train":
            state["dy"] = (0.1 * normal(n, c, *space)).to(dtype).contiguous(memory_format=fmt)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
        return state
    # gradients lie one behind the other in a flat buffer, as the buckets of data-parallel training have them; so do the weights
    # and the optimiser's states here, so that a pass can return them whole
    shapes = _NETS[case["net"]](case["nf"])
    total = sum(math.prod(s) for s in shapes)
    grads = (0.01 * normal(total) * (0.1 + normal(total).square())).to(dtype)       # heavy-tailed, as gradients are
    state = {"case": case, "flat": grads, "grads": _views(grads, shapes)}
    if case["op"] == "adam":
        flat = {"p": (0.05 * normal(total)).to(dtype), "m": 0.005 * normal(total), "v": 1e-5 * (0.01 + normal(total).square())}
        state["flats"] = flat
        state.update({k: _views(t, shapes) for k, t in flat.items()})
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return {"gn": _run_gn, "gn_train": _run_gn_train, "norm": _run_norm, "clip": _run_clip, "adam": _run_adam}[state["case"]["op"]](state)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, 0.01 * z)
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def _act_slope(z, act):
    if act in ("relu", "leaky_relu"):
        return torch.where(z > 0, 1.0, 0.01 if act == "leaky_relu" else 0.0)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _normalised(x, groups):
    """(x - mean) / deviation in 64 bits, [n, groups, channels of the group, space...], and 1 / deviation"""
    xg = x.double().unflatten(1, (groups, -1))
    dims = tuple(range(2, xg.dim()))
    mean = xg.mean(dims, keepdim=True)
    rstd = 1 / torch.sqrt((xg - mean).square().mean(dims, keepdim=True) + EPS)
    return (xg - mean) * rstd, rstd


def _per_channel(v, like):
    return v.view([1, -1] + [1] * (like.dim() - 2))


@torch.no_grad()
def _plain_gn(state, train):
    case, x, w, b = state["case"], state["x"], state["weight"], state["bias"]
    hat, rstd = _normalised(x, case["groups"])
    z = hat.flatten(1, 2) * _per_channel(w, x) + _per_channel(b, x)
    y = _act(z.float(), case["act"]).to(x.dtype)
    if not train:
        return y
    side = z if case["act"] in ("relu", "leaky_relu") else z.float()
    dz = state["dy"].float() * _act_slope(side, case["act"]).float()
    others = [0] + list(range(2, x.dim()))
    db = dz.sum(others, dtype=torch.float64)
    dw = (dz * hat.flatten(1, 2)).sum(others)
    dh = (dz * _per_channel(w, x)).unflatten(1, (case["groups"], -1))
    dims = tuple(range(2, dh.dim()))
    mean1 = dh.mean(dims, keepdim=True, dtype=torch.float64)
    mean2 = (dh * hat).mean(dims, keepdim=True)
    dx = (rstd * (dh - mean1 - hat * mean2)).flatten(1, 2)
    return y, dx.to(x.dtype), dw.float(), db.float()


def _run_gn(state):
    if own:
        from genre_shapehd_amd import group_norm_act
        return group_norm_act(state["x"], state["case"]["groups"], state["weight"], state["bias"], eps=EPS, act=state["case"]["act"], slope=0.01)
    return _plain_gn(state, False)


def _run_gn_train(state):
    if own:
        from genre_shapehd_amd import group_norm_act
        leaves = state["x"], state["weight"], state["bias"]
        y = group_norm_act(leaves[0], state["case"]["groups"], leaves[1], leaves[2], eps=EPS, act=state["case"]["act"], slope=0.01)
        return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))
    return _plain_gn(state, True)


def _plain_norm(grads, kind):
    if kind == "inf":
        return torch.stack([g.abs().max() for g in grads]).max().float()
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()


def _plain_factor(grads, case):
    norm = _plain_norm(grads, case["norm"])
    return norm, (case["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)


def _run_norm(state):
    if own:
        from genre_shapehd_amd import grad_norm
        return grad_norm(state["grads"], norm_type=float(state["case"]["norm"]))
    return _plain_norm(state["grads"], state["case"]["norm"])


def _run_clip(state):
    case = state["case"]
    if own:
        from genre_shapehd_amd import clip_grads_
        norm = clip_grads_(state["grads"], case["max_norm"], norm_type=float(case["norm"]))
    else:
        norm, factor = _plain_factor(state["grads"], case)
        [g.copy_(g.float() * factor) for g in state["grads"]]
    return norm, state["flat"]


def _plain_adam(p, g, m, v, factor, case):
    g = g.float() * factor + case["decay"] * p.float()
    m.copy_(BETA1 * m + (1 - BETA1) * g)
    v.copy_(BETA2 * v + (1 - BETA2) * g * g)
    root = torch.sqrt(v) / math.sqrt(1 - BETA2 ** case["step"]) + ADAM_EPS
    p.copy_(p.float() - (LR / (1 - BETA1 ** case["step"])) * m / root)


def _run_adam(state):
    case = state["case"]
    if own:
        from genre_shapehd_amd import clip_adam_step_
        norm = clip_adam_step_(state["p"], state["grads"], state["m"], state["v"], case["step"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                               weight_decay=case["decay"], max_norm=case["max_norm"])
    else:
        norm, factor = _plain_factor(state["grads"], case)
        [_plain_adam(*t, factor, case) for t in zip(state["p"], state["grads"], state["m"], state["v"])]
    return norm, state["flats"]


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"].startswith("gn"):
        total = case["n"] * case["c"] * case["d"] * case["h"] * case["w"]
        if case["op"] == "gn":                                            # x in, y out; two sums, a product and a sum, the activation
            return {"bytes": 2 * size * total, "flops": 8 * total}
        return {"bytes": 4 * size * total, "flops": 24 * total}           # x and dy in, y and dx out
    total = sum(math.prod(s) for s in _NETS[case["net"]](case["nf"]))
    if case["op"] == "norm":
        return {"bytes": size * total, "flops": 2 * total}
    if case["op"] == "clip":
        return {"bytes": 2 * size * total, "flops": 3 * total}
    return {"bytes": (3 * size + 16) * total, "flops": 16 * total}        # p, g, m, v in; p, m, v out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"].startswith("gn"):
        return _exact_gn(case, state)
    g = state["flat"].double()
    norm = g.abs().amax() if case["norm"] == "inf" else torch.linalg.vector_norm(g)
    if case["op"] == "norm":
        return norm
    g = g * min(1.0, case["max_norm"] / (float(norm) + CLIP_EPS))
    if case["op"] == "clip":
        return norm, g
    p, m, v = (state["flats"][k].double() for k in "pmv")
    g = g + case["decay"] * p
    m = m.lerp(g, 1 - BETA1)
    v = v.lerp(g.pow(2), 1 - BETA2)
    m_hat, v_hat = m / (1 - BETA1 ** case["step"]), v / (1 - BETA2 ** case["step"])
    return norm, {"p": p - LR * m_hat / (v_hat.pow(0.5) + ADAM_EPS), "m": m, "v": v}


def _exact_gn(case, state):
    """the forward definition on the values as they lie in one long row per group, and its gradients by automatic differentiation"""
    x, w, b = (state[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias"))
    rows = x.reshape(case["n"] * case["groups"], -1)
    var, mean = torch.var_mean(rows, 1, keepdim=True, correction=0)
    hat = ((rows - mean) / (var + EPS).sqrt()).reshape(case["n"], case["c"], -1)
    z = hat * w[:, None] + b[:, None]
    y = {"none": lambda t: t, "relu": lambda t: t * (t > 0), "leaky_relu": lambda t: t * ((t > 0) + 0.01 * (t <= 0)),
         "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z).reshape(x.shape)
    if case["op"] == "gn":
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), state["dy"].double()))
