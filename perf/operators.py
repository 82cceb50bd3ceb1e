"""The operators of the 4-bit caches: what is measured of them.

The cache of the global layers and the caches of the camera head can be held in 4 bits.  A row of `head_dim` values is cut into
blocks of 16; a block is stored as one 8-bit scale s and sixteen 4-bit values c, and stands for s * c:
    s  five exponent and three mantissa bits, no sign: max|x| / 6 rounded to the nearest (ties to even), at most 10240
    c  0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives: x / s rounded to the nearest (ties to even), at most 6
K and V are rounded to bf16 before (as the cache in 16 bits holds them) where the cache of the global layers takes them, and taken
in fp32 by the camera head's.

Operators
  append     a frame's rows go into the paged cache.  "qkv": from the output of the qkv Linear layer, with the norms of queries and
             keys for each head and the position rotation on the way; "kv": from finished K and V.  The rows are read back as the
             values they stand for (c and s), and taken out again, so that the cache is the same before every pass.
  attention  softmax(q k^T / 8) v over the visible pages of the cache: patches of the anchor frames and of the window, special
             tokens of all frames.
  step       a streamed frame that is no keyframe: append from qkv, attention of the frame's queries, and the frame out again.
  decode     the camera head: one token a frame, attention of `new` tokens over the cached ones and each other; with `store` their
             rows are appended, read back and taken out again.

Lengths and sizes are those of the models behind this backend: frames of 518 x (252 ... 518) and of 182 pixels on a side (patch
14), six special tokens, heads of 64 (the camera head's 128), caches of 1 ... 10,000 frames.
"""
import math

import torch

own = False

DEV = "cuda"
SPECIAL = 6                    # camera, register and scale tokens of a frame
BLOCK = 16                     # values of a block


def listed():
    return [
        # one frame at 518 x 378 through one global layer, bf16 under autocast: the append of every streamed frame
        dict(name="append_frame", op="append", source="qkv", pph=27, ppw=37, heads=16, src="bf16", norm=True, rope="3d"),
        # a frame of the small test model in fp32 (126 x 182 pixels): launches count
        dict(name="append_small_f32", op="append", source="qkv", pph=9, ppw=13, heads=16, src="f32", norm=True, rope="2d"),
        # finished K and V of a frame (phase 1, compiled blocks), an odd number of heads
        dict(name="append_kv", op="append", source="kv", pph=18, ppw=37, heads=3, src="bf16", norm=False, rope="none"),
        # the headline workload: a frame's queries over a 10,000-frame cache (131,928 tokens)
        dict(name="attn_10k", op="attention", pph=27, ppw=37, heads=16, cached=10000, scale=8, window=64, n_q=1005, src="bf16", lse=False),
        # the same at the trained context of 320 frames (window full, 73,848 tokens)
        dict(name="attn_320", op="attention", pph=27, ppw=37, heads=16, cached=320, scale=8, window=64, n_q=1005, src="bf16", lse=False),
        # the first frames after the scale pass: short cache
        dict(name="attn_start", op="attention", pph=27, ppw=37, heads=16, cached=9, scale=8, window=64, n_q=1005, src="bf16", lse=False),
        # one query token over the long cache: a stream over the pages
        dict(name="attn_token_10k", op="attention", pph=27, ppw=37, heads=16, cached=10000, scale=8, window=64, n_q=1, src="bf16", lse=False),
        # the special tokens alone over an anchor frame, a window of 16 and 1,000 frames of memory, fp32 queries, with the log-sum-exp
        dict(name="attn_special", op="attention", pph=27, ppw=37, heads=16, cached=1017, scale=1, window=16, n_q=6, src="f32", lse=True),
        # a streamed frame of the small test model: append and attention over a short window
        dict(name="step_small", op="step", pph=9, ppw=13, heads=16, cached=40, scale=2, window=8, src="bf16"),
        # the camera head at 10,000 cached frames, and at the start of a sequence (the smallest call)
        dict(name="decode_10k", op="decode", heads=16, head_dim=128, cached=10000, new=1, store=False),
        dict(name="decode_start", op="decode", heads=16, head_dim=128, cached=12, new=1, store=True),
        # several frames at once (a chunk of a sequence that starts behind a long one), heads of 64
        dict(name="decode_8", op="decode", heads=3, head_dim=64, cached=2001, new=8, store=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "step", "decode", "decode"])
    # square and wide frames with a long side of 518 or of the small model's 182 pixels, either way up
    pph, ppw = rng.choice([(rng.randint(18, 37), 37), (37, rng.randint(18, 36)), (rng.randint(7, 13), 13), (rng.randint(3, 30), rng.randint(3, 36))])
    heads = rng.choice([16, 16, 16, 1, 2, 3, 12])
    src = rng.choice(["bf16", "bf16", "f32"])
    if op == "append":
        source = rng.choice(["qkv", "qkv", "kv"])
        return dict(op=op, source=source, pph=pph, ppw=ppw, heads=heads, src=src, norm=source == "qkv" and rng.random() < 0.8,
                    rope=rng.choice(["3d", "3d", "2d", "none"]) if source == "qkv" else "none")
    if op == "decode":
        new = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 20)])
        return dict(op=op, heads=rng.choice([16, 16, 2, 3]), head_dim=rng.choice([128, 128, 64]), cached=_log(rng, 1, 10000), new=new,
                    store=rng.random() < 0.5)
    scale, window = rng.choice([(8, 64), (8, 64), (1, 16), (2, 8), (rng.randint(1, 8), rng.randint(2, 64))])
    tokens = pph * ppw + SPECIAL
    cached = _log(rng, 1, 10000)
    frames = min(cached, scale + window)
    while tokens * (frames * pph * ppw + cached * SPECIAL) * heads > 1005 * 131928 * 16:      # no more than the largest listed case
        cached = cached * 3 // 4
        window = max(2, window * 3 // 4)
        frames = min(cached, scale + window)
    if op == "step":
        return dict(op=op, pph=pph, ppw=ppw, heads=heads, cached=cached, scale=scale, window=window, src=src)
    n_q = rng.choice([tokens, tokens, 1, SPECIAL, _log(rng, 1, tokens)])
    return dict(op=op, pph=pph, ppw=ppw, heads=heads, cached=cached, scale=scale, window=window, n_q=n_q, src=src, lse=rng.random() < 0.3)


# ---- inputs ------------------------------------------------------------------------------------------------

def _visible_frames(case):
    """(patch frames that are visible, of the cache as it stands before the pass)"""
    anchors = min(case["cached"], case["scale"])
    return anchors, min(max(case["cached"] - case["scale"], 0), case["window"])


def _raw(case, seed):
    """The tensors of a case, from its seed: both sides and exact() start from these."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    dtype = {"bf16": torch.bfloat16, "f32": torch.float32}
    r = {}
    if case["op"] == "decode":
        H, D = case["heads"], case["head_dim"]
        channels = 0.4 * rand(H, D).exp()                     # some channels of V are louder than others
        r["k"], r["v"] = rand(case["cached"], H, D), rand(case["cached"], H, D) * channels
        r["q"], r["k_new"], r["v_new"] = rand(case["new"], H, D), rand(case["new"], H, D), rand(case["new"], H, D) * channels
        return r
    H, patches = case["heads"], case["pph"] * case["ppw"]
    tokens = patches + SPECIAL
    src = dtype[case["src"]]
    if case["op"] in ("append", "step"):
        if case["op"] == "step" or case["source"] == "qkv":
            loud = 1 + 0.5 * rand(3 * H * 64).abs()
            r["qkv"] = (rand(tokens, 3 * H * 64) * loud).to(src)
            with_norm = case["op"] == "step" or case["norm"]
            r["norm"] = tuple(x for _ in range(2) for x in (1 + 0.1 * rand(64), 0.1 * rand(64))) if with_norm else None
            rope = "3d" if case["op"] == "step" else case["rope"]
            r["cs"] = None if rope == "none" else _table(case, rope)
            r["rope"] = rope
        else:
            r["k"], r["v"] = rand(tokens, H, 64).to(src), (rand(tokens, H, 64) * 0.4 * rand(H, 64).exp()).to(src)
    if case["op"] in ("attention", "step"):
        anchors, recent = _visible_frames(case)
        channels = 0.4 * rand(H, 64).exp()
        r["k_patch"], r["v_patch"] = rand(anchors + recent, patches, H, 64).bfloat16(), (rand(anchors + recent, patches, H, 64) * channels).bfloat16()
        r["k_special"], r["v_special"] = rand(case["cached"], SPECIAL, H, 64).bfloat16(), (rand(case["cached"], SPECIAL, H, 64) * channels).bfloat16()
    if case["op"] == "attention":
        r["q"] = rand(case["n_q"], H, 64).to(src)
    return r


def _table(case, rope):
    """cos and sin [tokens, 32, 2] fp32.  3-D: frame 5; ten, eleven and eleven frequencies for time, height and width.  2-D: sixteen each
    for height and width."""
    pph, ppw = case["pph"], case["ppw"]
    f64 = dict(dtype=torch.float64, device=DEV)
    i = torch.arange(pph * ppw, device=DEV)
    special = torch.arange(SPECIAL, **f64)
    if rope == "3d":
        y, x = torch.cat([special, SPECIAL + (i // ppw).double()]), torch.cat([special, SPECIAL + (i % ppw).double()])
        inv = lambda n: 10000.0 ** (-torch.arange(n, **f64) / n)
        angle = torch.cat([(5.0 * inv(10)).expand(len(y), 10), y[:, None] * inv(11), x[:, None] * inv(11)], dim=1)
    else:
        zero = torch.zeros(SPECIAL, **f64)
        y, x = torch.cat([zero, (i // ppw + 1).double()]), torch.cat([zero, (i % ppw + 1).double()])
        inv = 100.0 ** (-torch.arange(16, **f64) / 16)
        angle = torch.cat([y[:, None] * inv, x[:, None] * inv], dim=1)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


def _visible(r):
    """K and V in the order of the visible pages: [tokens, H, 64] bf16."""
    flat = lambda t: t.reshape(-1, t.shape[-2], 64)
    return (torch.cat([flat(r["k_patch"]), flat(r["k_special"])]), torch.cat([flat(r["v_patch"]), flat(r["v_special"])]))


def prepare(case, seed):
    r = _raw(case, seed)
    state = {"case": case}
    for name in ("q", "qkv", "norm", "cs", "rope", "k_new", "v_new"):
        if name in r:
            state[name] = r[name]
    if case["op"] == "append" and "k" in r:
        state["k"], state["v"] = r["k"], r["v"]
    if own:
        state["cache"] = _own_cache(case, r)
    elif case["op"] in ("attention", "step"):
        k, v = _visible(r)
        state["k_cache"], state["v_cache"] = _quantise(k), _quantise(v)
    elif case["op"] == "decode":
        state["k_cache"], state["v_cache"] = _quantise(r["k"]), _quantise(r["v"])
    return state


def _own_cache(case, r):
    import lingbot_map_b200 as P
    H = case["heads"]
    if case["op"] == "decode":
        cache = P.DecodeCache(H, case["head_dim"], DEV, capacity=case["cached"] + case["new"], kv_bits=4)
        cache.append(r["k"], r["v"])
        return cache
    tokens = case["pph"] * case["ppw"] + SPECIAL
    scale, window, cached = case.get("scale", 1), case.get("window", 1), case.get("cached", 0)
    m = P.B200KVCacheManager(1, scale + window + 16, tokens, H, 64, device=DEV, num_special_tokens=SPECIAL, scale_frames=scale,
                             sliding_window=window, max_total_frames=cached + 2, kv_bits=4)
    if not cached:
        return m
    anchors, recent = _visible_frames(case)
    k, v = torch.empty(tokens, H, 64, dtype=torch.bfloat16, device=DEV), torch.empty(tokens, H, 64, dtype=torch.bfloat16, device=DEV)
    for f in range(cached):
        at = f if f < anchors else max(f - (cached - recent) + anchors, 0)      # patches of frames that will be evicted: any
        k[:SPECIAL], v[:SPECIAL], k[SPECIAL:], v[SPECIAL:] = r["k_special"][f], r["v_special"][f], r["k_patch"][at], r["v_patch"][at]
        m.append_frame(0, k, v)
        m.evict_frames(0, scale, window)
    return m


# ---- one pass ----------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(case, state)


def _run_own(case, s):
    from lingbot_map_b200 import _lib
    cache = s["cache"]
    if case["op"] == "decode":
        out = cache.attend(s["q"], s["k_new"], s["v_new"], case["store"])
        if not case["store"]:
            return {"out": out}
        rows = cache.rows_fp4(case["cached"], case["new"])
        cache.truncate(case["cached"])
        return {"out": out, "rows": rows}
    if case["op"] == "attention":
        return cache.compute_attention(0, s["q"], return_lse=case["lse"])
    mode = {"3d": _lib.ROPE_3D, "2d": _lib.ROPE_2D, "none": _lib.ROPE_NONE}
    norm = s.get("norm") or (None,) * 4
    if case["op"] == "step":
        q = cache.append_frame_fused(0, s["qkv"], *norm, s["cs"], mode[s["rope"]])
        out = cache.compute_attention(0, q)
        cache.rollback_last_frame(0)
        return {"q": q, "out": out}
    if case["source"] == "qkv":
        q = cache.append_frame_fused(0, s["qkv"], *norm, s["cs"], mode[s["rope"]])
    else:
        q = None
        cache.append_frame(0, s["k"], s["v"])
    rows = cache.last_frame_fp4(0)
    cache.rollback_last_frame(0)
    return {"q": q, "rows": rows}


def _quantise(x):
    """(values c, as float8 numbers that hold them, scales s, as float16 numbers that hold them) of rows of blocks of 16."""
    x = x.float()
    b = x.unflatten(-1, (-1, BLOCK))
    f = b.abs().amax(-1, keepdim=True) / 6
    step = torch.exp2(torch.frexp(f).exponent.clamp(min=-13).float() - 4)
    s = (torch.round(f / step) * step).clamp(max=10240.0)
    a = torch.where(s > 0, b / s, torch.zeros_like(b)).clamp(-6.0, 6.0)
    grid = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    c = torch.round(a / grid) * grid
    return c.flatten(-2).to(torch.float8_e4m3fn), s.squeeze(-1).half()


def _values(cs):
    c, s = cs
    return (c.float().unflatten(-1, (-1, BLOCK)) * s.float()[..., None]).flatten(-2)


def _norm_plain(x, w, b):
    x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w + b


def _rotate_plain(x, cs, rope):
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if rope == "3d":                                     # pairs (2m, 2m + 1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    x = x.unflatten(-1, (2, 2, 16))                      # halves; in each the pair (j, j + 16)
    a, b, c, s = x[..., 0, :], x[..., 1, :], c.unflatten(-1, (2, 16)), s.unflatten(-1, (2, 16))
    return torch.stack([a * c - b * s, a * s + b * c], dim=-2).flatten(-3)


def _qkv_plain(case, s):
    """q in bf16, K and V as they enter the cache."""
    q, k, v = s["qkv"].float().unflatten(-1, (3, case["heads"], 64)).unbind(1)
    if s["norm"] is not None:
        q, k = _norm_plain(q, *s["norm"][:2]), _norm_plain(k, *s["norm"][2:])
    if s["cs"] is not None:
        q, k = _rotate_plain(q, s["cs"], s["rope"]), _rotate_plain(k, s["cs"], s["rope"])
    return q.bfloat16(), _quantise(k.bfloat16()), _quantise(v.bfloat16())


def _attend_plain(q, k, v):
    """[n, H, D] fp32 each: softmax(q k^T / sqrt(D)) v and the log-sum-exp [n, H]."""
    x = torch.matmul(q.transpose(0, 1) * q.shape[-1] ** -0.5, k.permute(1, 2, 0))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x, v.transpose(0, 1)) / total
    return out.transpose(0, 1), (top + torch.log(total)).squeeze(-1).transpose(0, 1)


def _run_plain(case, s):
    if case["op"] == "decode":
        new = _quantise(s["k_new"]), _quantise(s["v_new"])
        k, v = torch.cat([_values(s["k_cache"]), _values(new[0])]), torch.cat([_values(s["v_cache"]), _values(new[1])])
        out = _attend_plain(s["q"], k, v)[0]
        return {"out": out, "rows": new[0] + new[1]} if case["store"] else {"out": out}
    if case["op"] == "attention":
        out, lse = _attend_plain(s["q"].bfloat16().float(), _values(s["k_cache"]), _values(s["v_cache"]))
        return (out.bfloat16(), lse) if case["lse"] else out.bfloat16()
    if case["op"] == "append" and case["source"] == "kv":
        q, k, v = None, _quantise(s["k"].bfloat16()), _quantise(s["v"].bfloat16())
    else:
        q, k, v = _qkv_plain(case, s)
    if case["op"] == "append":
        return {"q": q, "rows": k + v}
    out = _attend_plain(q.float(), torch.cat([_values(s["k_cache"]), _values(k)]), torch.cat([_values(s["v_cache"]), _values(v)]))[0]
    return {"q": q, "out": out.bfloat16()}


# ---- work --------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "decode":
        H, D, n, old = case["heads"], case["head_dim"], case["new"], case["cached"]
        row = H * (D // 2 + D // BLOCK)
        read_back = 2 * n * (row + H * (D + 2 * D // BLOCK)) if case["store"] else 0
        return {"bytes": 2 * old * row + 4 * n * H * D * 4 + read_back, "flops": 4 * n * (old + n) * H * D}
    H, patches = case["heads"], case["pph"] * case["ppw"]
    tokens, row = patches + SPECIAL, H * 36
    esz = 2 if case["src"] == "bf16" else 4
    if case["op"] == "attention":
        kv = sum(_visible_frames(case)) * patches + case["cached"] * SPECIAL
        return {"bytes": 2 * kv * row + case["n_q"] * H * (64 * (esz + 2) + (4 if case["lse"] else 0)), "flops": 4 * case["n_q"] * kv * H * 64}
    if case["op"] == "step":
        kv = sum(_visible_frames(case)) * patches + case["cached"] * SPECIAL + tokens
        return {"bytes": 2 * kv * row + 2 * tokens * row + tokens * H * 64 * (3 * esz + 4) + tokens * 256, "flops": 4 * tokens * kv * H * 64}
    parts = 3 if case["source"] == "qkv" else 2
    table = 0 if case["rope"] == "none" else tokens * 256
    return {"bytes": parts * tokens * H * 64 * esz + table + (parts - 2) * tokens * H * 128 + 2 * tokens * row + 2 * tokens * H * (64 + 8),
            "flops": 40 * tokens * H * 64}


# ---- the definition in 64 bits -----------------------------------------------------------------------------

def _grid_scales():
    """All scales in order: 0, the eight steps of 2^-17 below 2^-14, then eight to a power of two."""
    low = [k * 2.0 ** -17 for k in range(8)]
    high = [(1 + k / 8) * 2.0 ** e for e in range(-14, 14) for k in range(8)]
    return torch.tensor([x for x in low + high if x <= 10240.0], dtype=torch.float64, device=DEV)


def _nearest(x, grid):
    """Index of the nearest of the ordered values of `grid`, of two equally near the one with the even index."""
    mid = (grid[1:] + grid[:-1]) / 2
    below, above = torch.bucketize(x, mid, right=False), torch.bucketize(x, mid, right=True)
    return torch.where(below % 2 == 0, below, above)


def _exact_quantised(x):
    x = x.double()
    shape = x.shape
    x = x.reshape(*shape[:-1], shape[-1] // 16, 16)
    scales, steps = _grid_scales(), torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    s = scales[_nearest(x.abs().max(-1).values / 6, scales)]
    safe = torch.where(s > 0, s, torch.ones_like(s))[..., None]
    c = torch.where(s[..., None] > 0, steps[_nearest(x.abs() / safe, steps)] * torch.sign(x), torch.zeros_like(x))
    return c.reshape(shape), s


def _exact_values(c, s):
    return c * s.repeat_interleave(16, dim=-1)


def _exact_attention(q, k, v):
    q, out, lse = q.double(), [], []
    for h in range(q.shape[1]):
        logits = (q[:, h] @ k[:, h].T) / math.sqrt(q.shape[-1])
        total = torch.logsumexp(logits, -1)
        out.append(torch.exp(logits - total[:, None]) @ v[:, h])
        lse.append(total)
    return torch.stack(out, 1), torch.stack(lse, 1)


def _exact_frame(case, r):
    H, tokens = case["heads"], case["pph"] * case["ppw"] + SPECIAL
    parts = r["qkv"].double().view(tokens, 3, H, 64)
    done = []
    for i in range(2):
        x = parts[:, i]
        if r["norm"] is not None:
            w, b = r["norm"][2 * i].double(), r["norm"][2 * i + 1].double()
            centred = x - x.sum(-1, keepdim=True) / 64
            x = centred / torch.sqrt((centred ** 2).sum(-1, keepdim=True) / 64 + 1e-5) * w + b
        if r["cs"] is not None:
            turn = torch.view_as_complex(r["cs"].double())[:, None]
            if r["rope"] == "3d":
                x = torch.view_as_real(torch.view_as_complex(x.reshape(tokens, H, 32, 2).contiguous()) * turn).reshape(tokens, H, 64)
            else:
                z = torch.cat([torch.complex(x[..., :16], x[..., 16:32]), torch.complex(x[..., 32:48], x[..., 48:])], -1) * turn
                x = torch.cat([z.real[..., :16], z.imag[..., :16], z.real[..., 16:], z.imag[..., 16:]], -1)
        done.append(x)
    return done[0], _exact_quantised(done[1].bfloat16()), _exact_quantised(parts[:, 2].bfloat16())


def exact(case, seed):
    r = _raw(case, seed)
    if case["op"] == "decode":
        k, v, kn, vn = (_exact_quantised(r[x]) for x in ("k", "v", "k_new", "v_new"))
        values = lambda a, b: torch.cat([_exact_values(*a), _exact_values(*b)])
        out = _exact_attention(r["q"], values(k, kn), values(v, vn))[0]
        return {"out": out, "rows": kn + vn} if case["store"] else {"out": out}
    if case["op"] == "append" and case["source"] == "kv":
        q, k, v = None, _exact_quantised(r["k"].bfloat16()), _exact_quantised(r["v"].bfloat16())
    elif case["op"] != "attention":
        q, k, v = _exact_frame(case, r)
    if case["op"] == "append":
        return {"q": q, "rows": k + v}
    old = [_exact_values(*_exact_quantised(x)) for x in _visible(r)]
    if case["op"] == "attention":
        out, lse = _exact_attention(r["q"].bfloat16(), *old)
        return (out, lse) if case["lse"] else out
    new = [_exact_values(*x) for x in (k, v)]
    return {"q": q, "out": _exact_attention(q.bfloat16(), torch.cat([old[0], new[0]]), torch.cat([old[1], new[1]]))[0]}
