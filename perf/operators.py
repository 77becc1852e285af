"""Attention operators around the window attention, timed on their own.

Three kinds of call, all public entry points of ``ops``:

  qk      ``qk_norm_rope``: RMS norm of every query and key head and the position rotation, between the to_qkv projection and
          the attention
  cross   ``cross_attention``: grid tokens attend to an encoder's states (observations, another model's tokens), or a few
          places are read out of a whole grid
  prefix  ``cross_attention(prefix=...)``: the members of an ensemble share a context and have states of their own behind it

A case is a dict of plain values.  Heads are normalised before an attention like this one, so queries and keys are standard
normal values per component, and so are the values; input to ``qk_norm_rope`` is a projection's output of unit gain with some
heads louder than others.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False  # False: the operators in elementary torch operations; True: the framework's kernels

DEVICE = "cuda"
EPS = 1e-6
MAX_FLOPS = 1.08e12  # a drawn case costs no more than the largest listed ones
MAX_BYTES = 8.0e9
MAX_SCORES = 4.2e9


def _qk(name, tokens, heads, k_heads, head_dim, **kw):
    c = {"name": name, "kind": "qk", "tokens": tokens, "heads": heads, "k_heads": k_heads, "head_dim": head_dim, "layout": "planes",
         "x": "bf16", "gain": "bf16", "gain_per_head": False, "rotated": head_dim, "interleaved": False, "ws_y": 16, "ws_x": 16, "W": tokens,
         "batch": 1, "q_scale": 1.0}
    c.update(kw)
    return c


def _cross(kind, name, batch, queries, heads, kv_heads, head_dim, keys, **kw):
    c = {"name": name, "kind": kind, "batch": batch, "queries": queries, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "keys": keys, "prefix": 0, "kv_batch": batch, "ragged": 0.0, "empty": False, "masked": 0.0, "layout": "rows"}
    c.update(kw)
    return c


def listed():
    return [
        # The smallest call: the projected queries of four readout places, 12 heads of 128, one row of positions each.  Launch and host time.
        _qk("qk_readout_4", 4, 12, 0, 128, layout="rows", ws_y=4, ws_x=1, W=1),
        # The 1-degree block's queries and keys (8 heads of 64), as head planes on the way to 12 x 12 window attention, which wants
        # q multiplied by scale * log2(e).
        _qk("qk_180x360", 64800, 8, 8, 64, ws_y=12, ws_x=12, W=360, q_scale=0.125 * 1.4426950408889634),
        # ... and the full quarter-degree grid with 16 heads: the largest, 4.2 GB in and out.
        _qk("qk_720x1440", 1036800, 16, 16, 64, ws_y=16, ws_x=16, W=1440, q_scale=0.125 * 1.4426950408889634),
        # The reference's head form at an odd size: 3 heads of 128 out of the rows of one [tokens, 1152] matrix, two members, rectangular
        # windows, f32 gains per head, neighbouring columns rotated, and only the first half of them.
        _qk("qk_ref_rows", 12480, 3, 3, 128, layout="fused", gain="f32", gain_per_head=True, rotated=64, interleaved=True, ws_y=12, ws_x=8,
            W=104, batch=2),
        # A 32 x 64 grid attends to a short context: the smallest grid of this repository, launch time counts.
        _cross("cross", "cross_32x64", 1, 2048, 4, 4, 32, 77),
        # Two members on the 1-degree grid, each with its own number of observations, one in seven of which is missing.
        _cross("cross", "cross_180x360_masked", 2, 64800, 8, 8, 64, 1000, ragged=0.4, masked=0.15),
        # The full grid against 256 states: the largest by operations.
        _cross("cross", "cross_720x1440", 1, 1036800, 16, 16, 64, 256, layout="planes"),
        # One place is read out of the 1-degree grid of each of four members, 12 heads of 128: bound by reading the keys and values.
        _cross("cross", "cross_readout_1", 4, 1, 12, 12, 128, 64800),
        # 37 places against a 120 x 120 grid, grouped heads, lengths that end inside a tile, a member with no states at all.
        _cross("cross", "cross_readout_37", 5, 37, 8, 2, 64, 14400, ragged=0.9, empty=True),
        # Sixteen members, one query each: 16 384 shared states, up to 64 of their own.
        _cross("prefix", "prefix_single_16", 16, 1, 12, 12, 64, 64, prefix=16384, ragged=0.8),
        # Eight members read nine places, grouped heads of 128, from a shared 180 x 360 grid and 500 states of their own.
        _cross("prefix", "prefix_readout_9", 8, 9, 12, 4, 128, 500, prefix=64800, ragged=0.5),
        # Three members on a 60 x 104 grid attend to 1024 shared and up to 200 own states, 3 heads of 128.
        _cross("prefix", "prefix_grid_60x104", 3, 6240, 3, 3, 128, 200, prefix=1024, ragged=0.7, layout="planes"),
    ]


# ----------------------------------------------------------------------------------------------
# drawn cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qk", "cross", "cross", "prefix"])
    if kind == "qk":
        head_dim = rng.choice([32, 64, 64, 128])
        heads = _log_int(rng, 1, 24)
        k_heads = rng.choice([heads, heads, 0, math.gcd(heads, 4)])
        tokens = _log_int(rng, 1, 300000)
        case = _qk("", tokens, heads, k_heads, head_dim, layout=rng.choice(["planes", "rows", "fused"]), x=rng.choice(["bf16", "bf16", "f32"]),
                   gain=rng.choice(["bf16", "f32"]), gain_per_head=rng.random() < 0.4, rotated=rng.choice([head_dim, head_dim, head_dim // 2, 0]),
                   interleaved=rng.random() < 0.5, ws_y=_log_int(rng, 4, 60), ws_x=_log_int(rng, 4, 60), W=_log_int(rng, 4, 1440),
                   batch=rng.randint(1, 3), q_scale=rng.choice([1.0, head_dim ** -0.5]))
        while work(case)["bytes"] > MAX_BYTES:
            case["tokens"] //= 2
        del case["name"]
        return case
    head_dim = rng.choice([32, 64, 64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 3, 4])
    batch = rng.choice([1, 1, 2, 3, 4, 7, 16])
    if rng.random() < 0.5:  # a grid attends to a context
        queries, keys = _log_int(rng, 256, 129600), _log_int(rng, 1, 8192)
    else:  # a few places are read out of a grid
        queries, keys = _log_int(rng, 1, 256), _log_int(rng, 64, 129600)
    case = _cross(kind, "", batch, queries, heads, kv_heads, head_dim, keys, ragged=rng.choice([0.0, 0.5, 0.95]),
                  empty=batch > 1 and rng.random() < 0.25, masked=rng.choice([0.0, 0.0, 0.1, 0.6]), layout=rng.choice(["rows", "planes", "fused"]))
    if kind == "prefix":
        case["prefix"], case["keys"] = keys, _log_int(rng, 1, 512)
    elif rng.random() < 0.25:
        case["kv_batch"], case["ragged"], case["empty"] = 1, 0.0, False

    def too_much():
        w = work(case)
        scores = float(batch) * heads * case["queries"] * (case["prefix"] + case["keys"])
        kv = 2.0 * 2 * (case["prefix"] + case["keys"]) * batch * heads * head_dim
        return w["flops"] > MAX_FLOPS or w["bytes"] > MAX_BYTES or scores > MAX_SCORES or kv > MAX_BYTES

    while too_much():
        for n in ("queries", "keys", "prefix"):
            case[n] = case[n] if case[n] <= 1 else max(1, int(case[n] * 0.7))
    del case["name"]
    return case


# ----------------------------------------------------------------------------------------------
# inputs

def _lengths(case):
    """Keys of each member: from all of them down to (1 - ragged) of them, none for the last member of an "empty" case."""
    n, B = case["keys"], case["kv_batch"]
    out = [n - int(n * case["ragged"] * b / max(1, B - 1)) for b in range(B)]
    if case["empty"]:
        out[-1] = 0
    return out


def _rotation(case, positions, dim):
    """cos | sin of the angles, f32 [positions, rotated]: the first half of the pairs turns with the row, the other with the column."""
    pairs = dim // 2
    y, x = positions // case["ws_x"], positions % case["ws_x"]
    axis = (pairs + 1) // 2
    freq = 10000.0 ** (-torch.arange(axis, dtype=torch.float64, device=DEVICE) / axis)
    angle = torch.cat([y[:, None] * freq, x[:, None] * freq], dim=1)[:, :pairs]
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _prepare_qk(case, g):
    D, H, Hk = case["head_dim"], case["heads"], case["k_heads"]
    n, B = case["tokens"] // case["batch"] or 1, case["batch"] if case["tokens"] >= case["batch"] else 1
    T = n * B
    x_dtype = torch.bfloat16 if case["x"] == "bf16" else torch.float32
    parts = 3 * max(H, Hk) if case["layout"] == "fused" else H + Hk
    loud = 0.5 + 1.5 * torch.rand(parts, 1, generator=g, device=DEVICE)
    if case["layout"] == "planes":  # what the head-plane projection writes: [heads, tokens, head_dim]
        planes = (torch.randn(parts, T, D, generator=g, device=DEVICE) * loud[:, None]).to(x_dtype)
        q, k = planes[:H].permute(1, 0, 2), planes[H:H + Hk].permute(1, 0, 2)
    else:  # heads side by side in the rows of one matrix; "fused": with the values' columns behind them
        rows = (torch.randn(T, parts, D, generator=g, device=DEVICE) * loud).to(x_dtype)
        q, k = rows[:, :H], rows[:, H:H + Hk]
    gain_dtype = torch.bfloat16 if case["gain"] == "bf16" else torch.float32

    def gain(heads):
        shape = (heads, D) if case["gain_per_head"] else (D,)
        return (1.0 + 0.2 * torch.randn(shape, generator=g, device=DEVICE)).to(gain_dtype)

    state = {"q": q, "k": k if Hk else None, "q_gain": gain(H), "k_gain": gain(Hk) if Hk else None, "table": None, "positions": None,
             "interleaved": case["interleaved"], "q_scale": case["q_scale"]}
    if case["rotated"]:
        # the window position of every token of the grid, the same for all members
        t = torch.arange(n, device=DEVICE)
        Y, X = t // case["W"], t % case["W"]
        state["positions"] = ((Y % case["ws_y"]) * case["ws_x"] + X % case["ws_x"]).int()
        state["table"] = _rotation(case, torch.arange(case["ws_y"] * case["ws_x"], device=DEVICE), case["rotated"])
    return state


def _heads_tensor(case, shape, g):
    """[.., rows, heads, head_dim] bf16: rows of heads side by side, head planes, or the first part of rows twice as wide."""
    *lead, n, h, d = shape
    if case["layout"] == "planes":
        return torch.randn(*lead, h, n, d, generator=g, device=DEVICE).bfloat16().transpose(-3, -2)
    if case["layout"] == "fused":
        return torch.randn(*lead, n, 2 * h, d, generator=g, device=DEVICE).bfloat16()[..., :h, :]
    return torch.randn(*lead, n, h, d, generator=g, device=DEVICE).bfloat16()


def _prepare_cross(case, g):
    B, D = case["batch"], case["head_dim"]
    state = {"q": _heads_tensor(case, (B, case["queries"], case["heads"], D), g), "lengths": None, "mask": None, "prefix": None}
    kv = (case["kv_batch"], case["keys"], case["kv_heads"], D)
    state["k"], state["v"] = _heads_tensor(case, kv, g), _heads_tensor(case, kv, g)
    if case["ragged"] or case["empty"]:
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
        # what lies behind a member's last state was never written: it may be anything
        past = torch.arange(case["keys"], device=DEVICE)[None] >= state["lengths"][:, None]
        state["k"][past] = math.nan
        state["v"][past] = math.inf
    if case["masked"]:
        state["mask"] = torch.rand(case["kv_batch"], case["keys"], generator=g, device=DEVICE) >= case["masked"]
        state["v"][~state["mask"]] = math.nan
    if case["prefix"]:
        pre = (case["prefix"], case["kv_heads"], D)
        state["prefix"] = (_heads_tensor(case, pre, g), _heads_tensor(case, pre, g))
    return state


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = _prepare_qk(case, g) if case["kind"] == "qk" else _prepare_cross(case, g)
    state["kind"] = case["kind"]
    return state


# ----------------------------------------------------------------------------------------------
# one pass

def _plain_norm_rope(x, gain, table, positions, interleaved, scale):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gain.float()
    if table is not None:
        T, R = x.shape[0], table.shape[1]
        turn = table[positions.long()].repeat(T // positions.numel(), 1)[:, None]
        cos, sin = turn[..., :R // 2], turn[..., R // 2:]
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
        turned = (a * cos - b * sin, a * sin + b * cos)
        turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
        y = torch.cat([turned, y[..., R:]], dim=-1)
    return (y * scale).bfloat16()


def _plain_attention(q, k, v, lengths, mask, prefix):
    B, Nq, H, D = q.shape
    allowed = torch.ones(k.shape[:2], dtype=torch.bool, device=q.device)
    if lengths is not None:
        allowed = torch.arange(k.shape[1], device=q.device)[None] < lengths[:, None]
    if mask is not None:
        allowed = allowed & mask
    kf = torch.where(allowed[:, :, None, None], k.float(), 0.0)
    vf = torch.where(allowed[:, :, None, None], v.float(), 0.0)
    if prefix is not None:
        pk, pv = prefix
        kf = torch.cat([pk.float().expand(k.shape[0], *pk.shape), kf], dim=1)
        vf = torch.cat([pv.float().expand(k.shape[0], *pv.shape), vf], dim=1)
        allowed = torch.cat([allowed.new_ones(k.shape[0], pk.shape[0]), allowed], dim=1)
    Hk = kf.shape[2]
    rows = q.float().unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hk, group * Nq, D]
    s = torch.matmul(rows, kf.permute(0, 2, 3, 1).contiguous()) * D ** -0.5
    s = torch.where(allowed[:, None, None], s, -math.inf)
    s = s - s.amax(-1, keepdim=True).clamp_min(-1e30)  # (a member without any state: no maximum)
    p = s.exp()
    o = torch.matmul(p, vf.permute(0, 2, 1, 3).contiguous()) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.unflatten(2, (H // Hk, Nq)).permute(0, 3, 1, 2, 4).flatten(2, 3).bfloat16()


@torch.no_grad()
def run(state):
    if state["kind"] == "qk":
        q, k, table, positions = state["q"], state["k"], state["table"], state["positions"]
        if own:
            ops = importlib.import_module("aeris-gb_amd").ops
            yq, yk = ops.qk_norm_rope(q, k, state["q_gain"], state["k_gain"], rotation=table, positions=positions,
                                      interleaved=state["interleaved"], eps=EPS, q_scale=state["q_scale"])
        else:
            yq = _plain_norm_rope(q, state["q_gain"], table, positions, state["interleaved"], state["q_scale"])
            yk = None if k is None else _plain_norm_rope(k, state["k_gain"], table, positions, state["interleaved"], 1.0)
        return {"q": yq} if yk is None else {"q": yq, "k": yk}
    if own:
        ops = importlib.import_module("aeris-gb_amd").ops
        return ops.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], key_mask=state["mask"], prefix=state["prefix"])
    return _plain_attention(state["q"], state["k"], state["v"], state["lengths"], state["mask"], state["prefix"])


# ----------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_norm_rope(x, gain, table, positions, interleaved, scale):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    step = 1 << 16
    for h in range(x.shape[1]):
        g = (gain[h] if gain.dim() == 2 else gain).double()
        for t0 in range(0, x.shape[0], step):
            row = x[t0:t0 + step, h].double()
            row = row / (row.square().sum(-1, keepdim=True) / row.shape[-1] + EPS).sqrt() * g
            if table is not None:
                R = table.shape[1]
                t = torch.arange(t0, t0 + row.shape[0], device=x.device) % positions.numel()
                turn = table[positions[t].long()].double()
                turn = torch.complex(turn[:, :R // 2], turn[:, R // 2:])
                j = torch.arange(R // 2, device=x.device)
                ja, jb = (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)
                z = torch.complex(row[:, ja], row[:, jb]) * turn
                row[:, ja], row[:, jb] = z.real, z.imag
            out[t0:t0 + step, h] = row * scale
    return out


def _exact_attention(case, s):
    q, k, v = s["q"], s["k"], s["v"]
    B, Nq, H, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lengths = _lengths(case)
    for b in range(B):
        bk = b if k.shape[0] > 1 else 0
        keep = torch.arange(lengths[bk] if s["lengths"] is not None else k.shape[1], device=q.device)
        if s["mask"] is not None:
            keep = keep[s["mask"][bk, :keep.numel()]]
        for hk in range(k.shape[2]):
            kk, vv = k[bk, keep, hk].double(), v[bk, keep, hk].double()
            if s["prefix"] is not None:
                kk, vv = torch.cat([s["prefix"][0][:, hk].double(), kk]), torch.cat([s["prefix"][1][:, hk].double(), vv])
            if kk.shape[0] == 0:
                continue
            step = max(1, (1 << 28) // kk.shape[0])
            for h in range(hk * (H // k.shape[2]), (hk + 1) * (H // k.shape[2])):
                for n0 in range(0, Nq, step):
                    logits = q[b, n0:n0 + step, h].double() @ kk.T / math.sqrt(D)
                    out[b, n0:n0 + step, h] = (logits - torch.logsumexp(logits, -1, keepdim=True)).exp() @ vv
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "qk":
        return _exact_attention(case, s)
    out = {"q": _exact_norm_rope(s["q"], s["q_gain"], s["table"], s["positions"], s["interleaved"], s["q_scale"])}
    if s["k"] is not None:
        out["k"] = _exact_norm_rope(s["k"], s["k_gain"], s["table"], s["positions"], s["interleaved"], 1.0)
    return out


# ----------------------------------------------------------------------------------------------
# what one pass cannot do without

def work(case):
    D = case["head_dim"]
    if case["kind"] == "qk":
        elements = float(case["tokens"]) * (case["heads"] + case["k_heads"]) * D
        table = 4.0 * case["ws_y"] * case["ws_x"] * case["rotated"]
        return {"bytes": elements * ((2 if case["x"] == "bf16" else 4) + 2) + table, "flops": 8.0 * elements}
    B, Nq, H, Hk = case["batch"], case["queries"], case["heads"], case["kv_heads"]
    own_keys = sum(_lengths(case)) * (1.0 - case["masked"])
    pairs = float(Nq) * (B * case["prefix"] + own_keys * (B // case["kv_batch"]))
    kv = (case["prefix"] + own_keys) * Hk * D * 2 * 2
    return {"bytes": 2.0 * 2 * B * Nq * H * D + kv, "flops": 4.0 * pairs * H * D}
