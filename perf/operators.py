"""The operators of a packed and a stepwise Mamba mixer, as they are used, with their plain forms.

Packed batches hold sequences of different lengths back to back: ``[tokens, channels]`` rows, ``offsets [S + 1]``.

* the selective scan over a packed batch, for prompts (states kept in a cache) and for training (with its gradients)
* the selective scan of one token per sequence against the cached states
* the causal conv1d + SiLU in front of it over a packed batch, for prompts and for training
* the same convolution of one token per sequence against the cached windows

``run`` computes them with elementary torch operations where ``own`` is false, and calls the package where it is true.
"""
import math
import random

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------
def _scan(name, kind, tokens, sequences, channels, states, dtype, **more):
    case = {"name": name, "op": "scan", "kind": kind, "tokens": tokens, "sequences": sequences, "channels": channels,
            "states": states, "rank": max(1, channels // 32), "dtype": dtype, "ragged": kind != "step", "pad": 0,
            "carry": False}
    return {**case, **more}


def _conv(name, kind, tokens, sequences, channels, taps, dtype, **more):
    case = {"name": name, "op": "conv", "kind": kind, "tokens": tokens, "sequences": sequences, "channels": channels,
            "taps": taps, "dtype": dtype, "ragged": kind != "step", "pad": 0, "carry": False}
    return {**case, **more}


def listed():
    return [
        # one user's short history enters a Mamba4Rec of the shipped size (d_inner 128, d_state 256): latency counts
        _scan("scan prompt one short", "prompt", 37, 1, 128, 256, "f32"),
        # prompts of a serving batch, some of them the next piece of a longer prompt, behind them the padding of the buffer
        _scan("scan prompts ragged", "prompt", 24576, 48, 2048, 16, "bf16", pad=100),
        # one long document at the benchmark's channels and state size
        _scan("scan prompt one long", "prompt", 65536, 1, 2048, 16, "bf16"),
        # a training batch of Mamba4Rec: 128 histories of up to 200 items, d_state 256
        _scan("scan training histories", "train", 12800, 128, 128, 256, "f32"),
        # a training batch of long packed sequences whose states continue from and into the neighbouring pieces
        _scan("scan training long", "train", 32768, 11, 2048, 16, "bf16", carry=True),
        # one interaction of one user
        _scan("scan step one", "step", 1, 1, 128, 256, "f32"),
        # a decoding batch of a large mixer
        _scan("scan step large", "step", 512, 512, 4096, 16, "bf16"),
        # the prompts' convolution at the channels of the serving batch above
        _conv("conv prompts ragged", "prompt", 24576, 48, 2048, 4, "bf16", pad=100),
        # the histories' convolution in training
        _conv("conv training histories", "train", 12800, 128, 128, 4, "f32"),
        # the long sequences' convolution in training, odd taps
        _conv("conv training long", "train", 65536, 11, 4096, 3, "bf16", carry=True),
        _conv("conv step one", "step", 1, 1, 128, 4, "f32"),
        _conv("conv step large", "step", 512, 512, 4096, 4, "bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op, kind = rng.choice(["scan", "scan", "conv"]), rng.choice(["prompt", "train", "step"])
    dtype = rng.choice(["bf16", "f32"])
    channels = _log_int(rng, 32, 4096)
    if rng.random() < 0.7:
        channels = max(32, channels // 32 * 32)
    if op == "conv":
        case = _conv("", kind, 0, 0, channels, rng.randint(2, 4), dtype)
        most = 65536 * 4096 // channels
    else:
        states = rng.choice([16, 16, 32, 64, 128, 256, rng.randint(1, 256)])
        case = _scan("", kind, 0, 0, channels, states, dtype)
        most = (32768 if kind == "train" else 65536) * 2048 * 16 // (channels * states)
        case["rank"] = rng.randint(1, 128)
    if kind == "step":
        case["tokens"] = case["sequences"] = _log_int(rng, 1, max(1, min(1024, most // 32)))
    else:
        case["tokens"] = _log_int(rng, 1, max(1, min(65536, most)))
        case["sequences"] = _log_int(rng, 1, max(1, case["tokens"] // 8))
        case["ragged"] = rng.random() < 0.8
        case["pad"] = rng.choice([0, 0, 1, 77])
        case["carry"] = kind == "train" and rng.random() < 0.5
    del case["name"]
    most = max(_cost(c) for c in listed())
    while _cost(case) > most:
        case["tokens"] = case["tokens"] // 2
        case["sequences"] = case["tokens"] if kind == "step" else min(case["sequences"], case["tokens"])
    return case


def _cost(case):
    need = work(case)
    return max(need["bytes"], need["flops"] / 50)


def _lengths(case):
    """The same lengths for every seed: shares of an exponential distribution, some sequences empty."""
    n, tokens = case["sequences"], case["tokens"]
    if not case["ragged"]:
        return [tokens * (i + 1) // n - tokens * i // n for i in range(n)]
    rng = random.Random(n * 1000003 + tokens)
    share = [0.0 if n > 4 and rng.random() < 0.04 else rng.expovariate(1.0) + 0.02 for _ in range(n)]
    total, at, ends = sum(share) or 1.0, 0.0, []
    share[-1] += 0.0 if sum(share) else 1.0
    for s in share:
        at += s
        ends.append(min(tokens, int(round(tokens * at / total))))
    ends[-1] = tokens
    return [e - b for b, e in zip([0] + ends[:-1], ends)]


# ---- what a program has in hand ------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dtype, D, S = DTYPES[case["dtype"]], case["channels"], case["sequences"]
    rows = case["tokens"] + case["pad"]

    def randn(*shape, to=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(to)

    s = {"case": case, "train": case["kind"] == "train"}
    lengths = torch.tensor(_lengths(case))
    s["longest"] = max(1, int(lengths.max()))     # the plain form's number of doublings goes by it
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).int().cuda()
    xz = randn(rows, 2 * D, to=dtype)             # in_proj's output: x and the gate side by side
    slots = S + S // 4 + 1
    s["slots"] = torch.randperm(slots, generator=gen, device="cuda")[:S].int()
    s["resume"] = torch.rand(S, generator=gen, device="cuda") < 0.5
    if case["op"] == "conv":
        K = case["taps"]
        s["x"] = xz[:, :D]
        s["weight"] = ((torch.rand(D, 1, K, generator=gen, device="cuda") * 2 - 1) / math.sqrt(K)).to(dtype)
        s["bias"] = ((torch.rand(D, generator=gen, device="cuda") * 2 - 1) / math.sqrt(K)).to(dtype)
        s["cache"] = randn(slots, K - 1, D, to=dtype)
        if s["train"]:
            s["x"] = s["x"].detach().requires_grad_(True)
            s["weight"].requires_grad_(True), s["bias"].requires_grad_(True)
            s["start"] = randn(S, K - 1, D, to=dtype).requires_grad_(True) if case["carry"] else None
            s["grad"] = randn(rows, D, to=dtype)
            s["grad_end"] = randn(S, K - 1, D, to=dtype) if case["carry"] else None
        return s
    N, R = case["states"], case["rank"]
    proj = randn(rows, R + 2 * N, to=dtype)       # x_proj's output: dt_raw, B and C side by side
    s["u"] = torch.nn.functional.silu(randn(rows, D)).to(dtype)
    s["dt"] = (randn(rows, D) * 0.5).to(dtype)    # dt_proj's output without its bias
    s["B"], s["C"], s["z"] = proj[:, R:R + N], proj[:, R + N:], xz[:, D:]
    s["A"] = -torch.arange(1, N + 1, device="cuda").float() * torch.exp(0.1 * randn(D, N))
    step = torch.exp(torch.rand(D, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    s["bias"] = step + torch.log(-torch.expm1(-step))   # softplus(bias) lies in 0.001 .. 0.1
    s["D"] = 1 + 0.1 * randn(D)
    s["cache"] = 0.3 * randn(slots, D, N)
    if s["train"]:
        for name in ("u", "dt", "A", "B", "C", "z", "D", "bias"):
            s[name] = s[name].detach().requires_grad_(True)
        s["start"] = (0.3 * randn(S, D, N)).requires_grad_(True) if case["carry"] else None
        s["grad"] = randn(rows, D, to=dtype)
        s["grad_end"] = randn(S, D, N) if case["carry"] else None
    return s


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return (_plain_conv if s["case"]["op"] == "conv" else _plain_scan)(s)


def _run_own(s):
    from ossm_b200.mixer import causal_conv1d_silu_packed, causal_conv1d_silu_step
    from ossm_b200.selective_scan import selective_scan_packed, selective_scan_step

    kind = s["case"]["kind"]
    if s["case"]["op"] == "conv":
        if kind == "step":
            out = causal_conv1d_silu_step(s["x"], s["weight"], s["bias"], s["cache"], slots=s["slots"])
            return {"out": out, "cache": s["cache"]}
        if kind == "prompt":
            out = causal_conv1d_silu_packed(s["x"], s["weight"], s["bias"], s["offsets"], cache=s["cache"],
                                            slots=s["slots"], resume=s["resume"])
            return {"out": out, "cache": s["cache"]}
        out = causal_conv1d_silu_packed(s["x"], s["weight"], s["bias"], s["offsets"], initial_window=s["start"],
                                        return_window=s["start"] is not None)
        names = ["x", "weight", "bias"]
    else:
        common = {"delta_bias": s["bias"], "delta_softplus": True}
        args = (s["u"], s["dt"], s["A"], s["B"], s["C"])
        if kind == "step":
            out = selective_scan_step(*args, s["cache"], s["z"], s["D"], slots=s["slots"], **common)
            return {"out": out, "cache": s["cache"]}
        if kind == "prompt":
            out = selective_scan_packed(*args, s["offsets"], s["z"], s["D"], cache=s["cache"], slots=s["slots"],
                                        resume=s["resume"], **common)
            return {"out": out, "cache": s["cache"]}
        out = selective_scan_packed(*args, s["offsets"], s["z"], s["D"], initial_state=s["start"],
                                    return_state=s["start"] is not None, **common)
        names = ["u", "dt", "A", "B", "C", "z", "D", "bias"]
    outs, grads = (out,), (s["grad"],)
    if s["start"] is not None:
        outs, grads, names = out, (s["grad"], s["grad_end"]), names + ["start"]
    got = torch.autograd.grad(outs, [s[n] for n in names], grads)
    answer = {"grad_" + n: g for n, g in zip(names, got)}
    answer["out"] = outs[0].detach()
    if s["start"] is not None:
        answer["end"] = outs[1].detach()
    return answer


# ---- the plain forms -----------------------------------------------------------------------------
def _positions(s):
    """Rows that belong to a sequence, the sequence of each, and each one's place in it."""
    starts, ends = s["offsets"][:-1].long(), s["offsets"][1:].long()
    rows = torch.arange(s["case"]["tokens"] + s["case"]["pad"], device="cuda")
    seq = torch.bucketize(rows, ends, right=True).clamp(max=ends.numel() - 1)
    return starts, ends, seq, rows - starts[seq], rows < ends[-1]


def _start_state(s, zero):
    """What precedes each sequence, in 32 bits: the cached entry where it is resumed, what was given, or zeros."""
    if s["train"]:
        return zero if s["start"] is None else s["start"].float()
    return torch.where(s["resume"].view(-1, *[1] * (zero.dim() - 1)), s["cache"][s["slots"].long()].float(), zero)


def _doubling(a, b, longest):
    """``h[t] = a[t] h[t-1] + b[t]`` along the first axis, in place of ``b``, ``a`` zero where a sequence starts."""
    step = 1
    while step < longest:
        b[step:] += a[step:] * b[:-step]
        a[step:] = a[step:] * a[:-step]
        step *= 2
    return b


def _plain_scan(s):
    c = s["case"]
    u, z, Bm, Cm, A = s["u"].float(), s["z"].float(), s["B"].float(), s["C"].float(), s["A"]
    raw = s["dt"].float() + s["bias"]
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    gate = z / (1 + torch.exp(-z))
    if c["kind"] == "step":
        at = s["slots"].long()
        h = torch.exp(dt[:, :, None] * A) * s["cache"][at] + (dt * u)[:, :, None] * Bm[:, None, :]
        s["cache"][at] = h
        y = (h * Cm[:, None, :]).sum(-1) + s["D"] * u
        return {"out": (y * gate).to(s["u"].dtype), "cache": s["cache"]}
    starts, ends, seq, place, real = _positions(s)
    S, D, N = c["sequences"], c["channels"], c["states"]
    first = (place == 0) & real
    h0 = _start_state(s, torch.zeros(S, D, N, device="cuda"))
    decay = torch.exp(dt[:, :, None] * A)
    force = (dt * u)[:, :, None] * Bm[:, None, :]
    force[first] += decay[first] * h0[seq[first]]
    scale = decay if not s["train"] else decay.clone()
    scale[first] = 0
    h = _doubling(scale, force, s["longest"])
    y = torch.einsum("tdn,tn->td", h, Cm) + s["D"] * u
    out = (y * gate * real[:, None]).to(s["u"].dtype)
    filled = ends > starts
    last = (ends - 1).clamp(min=0)
    end = torch.where(filled[:, None, None], h[last], h0)
    if not s["train"]:
        s["cache"][s["slots"].long()] = end
        return {"out": out, "cache": s["cache"]}
    # the adjoint runs from each sequence's last row to its first
    g_out = s["grad"].float() * real[:, None]
    sig = 1 / (1 + torch.exp(-z))
    dy = g_out * gate
    dz = g_out * y * sig * (1 + z * (1 - sig))
    adj = dy[:, :, None] * Cm[:, None, :]
    if s["grad_end"] is not None:
        adj[last[filled]] += s["grad_end"][filled]
    back = torch.roll(decay, -1, 0)               # the decay of the row behind
    back[last[filled]] = 0
    back[~real] = 0
    adj = _doubling(back.flip(0), adj.flip(0), s["longest"]).flip(0)
    dB = torch.einsum("tdn,td->tn", adj, dt * u) * real[:, None]
    dC = torch.einsum("tdn,td->tn", h, dy)
    d_force = torch.einsum("tdn,tn->td", adj, Bm)
    before = torch.roll(h, 1, 0)
    before[first] = h0[seq[first]]
    d_arg = adj * before * decay                  # gradient of dt * A
    d_start = torch.where(filled[:, None, None], (adj * decay)[starts.clamp(max=place.numel() - 1)],
                          s["grad_end"] if s["grad_end"] is not None else torch.zeros_like(h0))
    dA = torch.einsum("tdn,td->dn", d_arg, dt * real[:, None])
    d_dt = torch.einsum("tdn,dn->td", d_arg, A) + d_force * u
    d_raw = (torch.where(raw > 20, d_dt, d_dt / (1 + torch.exp(-raw))) * real[:, None])
    du = (d_force * dt + dy * s["D"]) * real[:, None]
    answer = {"out": out, "grad_u": du.to(s["u"].dtype), "grad_A": dA,
              "grad_dt": d_raw.to(s["dt"].dtype), "grad_B": dB.to(s["B"].dtype), "grad_C": dC.to(s["C"].dtype),
              "grad_z": dz.to(s["z"].dtype), "grad_D": (dy * u).sum(0), "grad_bias": d_raw.sum(0)}
    if s["start"] is not None:
        answer |= {"grad_start": d_start, "end": end}
    return answer


def _plain_conv(s):
    c = s["case"]
    K, dtype, S, D = c["taps"], s["x"].dtype, c["sequences"], c["channels"]
    x, w, bias = s["x"].float(), s["weight"].float().view(D, K), s["bias"].float()
    if c["kind"] == "step":
        at = s["slots"].long()
        window = torch.cat([s["cache"][at].float(), x[:, None, :]], 1)
        pre = torch.einsum("bkd,dk->bd", window, w) + bias
        s["cache"][at] = window[:, 1:].to(dtype)
        return {"out": (pre / (1 + torch.exp(-pre))).to(dtype), "cache": s["cache"]}
    starts, ends, seq, place, real = _positions(s)
    rows = x.shape[0]
    before = _start_state(s, torch.zeros(S, K - 1, D, device="cuda"))
    # every sequence with its window in front, back to back: the row of token t is t + (K - 1) (seq + 1)
    long = torch.zeros(rows + (K - 1) * S + K, D, device="cuda")
    at = torch.where(real, torch.arange(rows, device="cuda") + (K - 1) * (seq + 1), rows + (K - 1) * S)
    front = (starts + (K - 1) * torch.arange(S, device="cuda"))[:, None] + torch.arange(K - 1, device="cuda")
    back = front + (ends - starts)[:, None]       # the last K - 1 rows of a sequence and its window
    long[front] = before
    long[at] = torch.where(real[:, None], x, 0.0)
    taps = at[:, None] - (K - 1) + torch.arange(K, device="cuda")
    seen = long[taps]                             # [rows, K, D]
    pre = torch.einsum("tkd,dk->td", seen, w) + bias
    sig = 1 / (1 + torch.exp(-pre))
    out = (pre * sig * real[:, None]).to(dtype)
    end = long[back]
    if not s["train"]:
        s["cache"][s["slots"].long()] = end.to(dtype)
        return {"out": out, "cache": s["cache"]}
    g = s["grad"].float() * real[:, None] * sig * (1 + pre * (1 - sig))
    g_long = torch.zeros_like(long)
    g_long.index_add_(0, taps.reshape(-1), torch.einsum("td,dk->tkd", g, w).reshape(-1, D))
    if s["grad_end"] is not None:
        g_long.index_add_(0, back.reshape(-1), s["grad_end"].float().reshape(-1, D))
    answer = {"out": out, "grad_x": (g_long[at] * real[:, None]).to(dtype),
              "grad_weight": torch.einsum("td,tkd->dk", g, seen).view(D, 1, K).to(dtype), "grad_bias": g.sum(0).to(dtype)}
    if s["start"] is not None:
        answer |= {"grad_start": g_long[front].to(dtype), "end": end.to(dtype)}
    return answer


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    e, D, S, T = (2 if case["dtype"] == "bf16" else 4), case["channels"], case["sequences"], case["tokens"]
    train, step = case["kind"] == "train", case["kind"] == "step"
    if case["op"] == "conv":
        K = case["taps"]
        window = S * (K - 1) * D * e
        read = T * D * e + D * (K + 1) * e
        if not train:
            return {"bytes": read + T * D * e + window * (2 if step else 1.5), "flops": T * D * (2 * K + 6)}
        # x and the two gradients, the output, the parameters' gradients, the windows and theirs
        return {"bytes": read + 3 * T * D * e + D * (K + 1) * e + (4 * window if case["carry"] else 0),
                "flops": T * D * (6 * K + 20)}
    N = case["states"]
    state = S * D * N * 4
    read = T * D * 3 * e + T * 2 * N * e + D * N * 4 + 2 * D * 4
    pairs = T * D * N
    if not train:
        # per state and step: the decay's argument and exponential, the forcing, the update, the output's sum
        return {"bytes": read + T * D * e + state * (2 if step else 1.5), "flops": 7 * pairs + 20 * T * D}
    return {"bytes": read + 5 * T * D * e + T * 2 * N * e + D * N * 4 + 2 * D * 4 + (4 * state if case["carry"] else 0),
            "flops": 25 * pairs + 60 * T * D}


# ---- the definition in 64 bits, step by step -------------------------------------------------------
def _walk(s):
    """The tokens' rows step by step: for each place the sequences that reach it (longest first) and their rows."""
    lengths, order = torch.tensor(_lengths(s["case"])).sort(descending=True, stable=True)
    starts = s["offsets"][:-1].long()[order.cuda()]
    ascending = (-lengths).contiguous()
    counts = torch.searchsorted(ascending, -torch.arange(1, s["longest"] + 1), right=True).tolist()
    return order.cuda(), starts, [n for n in counts if n > 0]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_conv if case["op"] == "conv" else _exact_scan)(s)


def _exact_scan(s):
    c, f = s["case"], torch.float64
    if c["kind"] == "step":
        s["offsets"], s["resume"] = torch.arange(c["sequences"] + 1, device="cuda").int(), torch.ones_like(s["resume"])
    u, Bm, Cm, A = s["u"].to(f), s["B"].to(f), s["C"].to(f), s["A"].to(f)
    dt = torch.nn.functional.softplus(s["dt"].to(f) + s["bias"].to(f))
    sig = torch.sigmoid(s["z"].to(f))
    order, starts, counts = _walk(s)
    S, D, N, rows = c["sequences"], c["channels"], c["states"], u.shape[0]
    start = torch.zeros(S, D, N, dtype=f, device="cuda")
    if s["train"]:
        start = start if s["start"] is None else s["start"].to(f)
    else:
        start[s["resume"]] = s["cache"].to(f)[s["slots"].long()][s["resume"]]
    h = start[order].clone()
    y = torch.zeros(rows, D, dtype=f, device="cuda")
    kept = torch.zeros(rows if s["train"] else 0, D, N, dtype=f, device="cuda")
    for t, n in enumerate(counts):
        at = starts[:n] + t
        if s["train"]:
            kept[at] = h[:n]
        h[:n] = torch.exp(dt[at].unsqueeze(-1) * A) * h[:n] + torch.einsum("sd,sn->sdn", dt[at] * u[at], Bm[at])
        y[at] = torch.einsum("sdn,sn->sd", h[:n], Cm[at]) + s["D"].to(f) * u[at]
    end = torch.zeros_like(h)
    end[order] = h
    if not s["train"]:
        cache = s["cache"].to(f)
        cache[s["slots"].long()] = end
        return {"out": y * s["z"].to(f) * sig, "cache": cache}
    dy = s["grad"].to(f) * s["z"].to(f) * sig
    du, ddt, dB, dC = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(Bm), torch.zeros_like(Cm)
    dA, dD = torch.zeros_like(A), torch.zeros(D, dtype=f, device="cuda")
    g = torch.zeros_like(h) if s["grad_end"] is None else s["grad_end"].to(f)[order].clone()
    for t in range(len(counts) - 1, -1, -1):
        n = counts[t]
        at = starts[:n] + t
        decay = torch.exp(dt[at].unsqueeze(-1) * A)
        state = decay * kept[at] + torch.einsum("sd,sn->sdn", dt[at] * u[at], Bm[at])
        dC[at] = torch.einsum("sdn,sd->sn", state, dy[at])
        g[:n] += torch.einsum("sd,sn->sdn", dy[at], Cm[at])
        forced = torch.einsum("sdn,sn->sd", g[:n], Bm[at])
        dB[at] = torch.einsum("sdn,sd->sn", g[:n], dt[at] * u[at])
        g[:n] *= decay
        through = g[:n] * kept[at]
        dA += torch.einsum("sdn,sd->dn", through, dt[at])
        ddt[at] = torch.einsum("sdn,dn->sd", through, A) + forced * u[at]
        du[at] = forced * dt[at] + dy[at] * s["D"].to(f)
        dD += (dy[at] * u[at]).sum(0)
    d_raw = ddt * -torch.expm1(-dt)
    zz = s["z"].to(f)
    in_use = torch.zeros(rows, 1, dtype=f, device="cuda")
    in_use[: c["tokens"]] = 1
    answer = {"out": y * zz * sig, "grad_u": du, "grad_dt": d_raw, "grad_A": dA, "grad_B": dB, "grad_C": dC,
              "grad_z": s["grad"].to(f) * y * sig * (1 + zz * (1 - sig)) * in_use, "grad_D": dD, "grad_bias": d_raw.sum(0)}
    if s["start"] is not None:
        d_start = torch.zeros_like(g)
        d_start[order] = g
        answer |= {"grad_start": d_start, "end": end}
    return answer


def _exact_conv(s):
    c, f = s["case"], torch.float64
    K, D, S, rows = c["taps"], c["channels"], c["sequences"], s["x"].shape[0]
    if c["kind"] == "step":
        s["offsets"], s["resume"] = torch.arange(S + 1, device="cuda").int(), torch.ones_like(s["resume"])
    x, w, bias = s["x"].detach().to(f), s["weight"].to(f).reshape(D, K), s["bias"].to(f)
    start = torch.zeros(S, K - 1, D, dtype=f, device="cuda")
    if s["train"]:
        start = start if s["start"] is None else s["start"].to(f)
    else:
        start[s["resume"]] = s["cache"].to(f)[s["slots"].long()][s["resume"]]
    ends = s["offsets"].tolist()
    out, gx = torch.zeros(rows, D, dtype=f, device="cuda"), torch.zeros(rows, D, dtype=f, device="cuda")
    end, gw, gb, gs = torch.zeros_like(start), torch.zeros_like(w), torch.zeros_like(bias), torch.zeros_like(start)
    for i in range(S):                            # one sequence after the other
        lo, hi = ends[i], ends[i + 1]
        seq = torch.cat([start[i], x[lo:hi]])
        n = hi - lo
        pre = bias + sum(w[:, k] * seq[k:k + n] for k in range(K))
        sig = torch.sigmoid(pre)
        out[lo:hi] = pre * sig
        end[i] = seq[n:]
        if s["train"]:
            g = s["grad"][lo:hi].to(f) * (sig + pre * sig * (1 - sig))
            d = torch.zeros_like(seq)
            for k in range(K):
                d[k:k + n] += w[:, k] * g
                gw[:, k] += (g * seq[k:k + n]).sum(0)
            if s["grad_end"] is not None:
                d[n:] += s["grad_end"][i].to(f)
            gb += g.sum(0)
            gs[i], gx[lo:hi] = d[:K - 1], d[K - 1:]
    if not s["train"]:
        cache = s["cache"].to(f)
        cache[s["slots"].long()] = end
        return {"out": out, "cache": cache}
    answer = {"out": out, "grad_x": gx, "grad_weight": gw.view(D, 1, K), "grad_bias": gb}
    if s["start"] is not None:
        answer |= {"grad_start": gs, "end": end}
    return answer
