"""The 4-bit caches on the GPU against the float64 oracle of the format (oracle/fp4_oracle.py).

What is stored is compared bit for bit.  Attention is compared with float64 softmax attention over the values that the cache stands for; the
bounds are derived at `bound_rows` and `bound_frame`."""
import numpy as np
import pytest
import torch

import lingbot_map_b200 as P
from lingbot_map_b200 import _lib
from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NS = 6


def dev(x, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV).to(dtype)


def bf(x):
    return torch.from_numpy(np.asarray(x, np.float32)).to(torch.bfloat16).float().numpy().astype(np.float64)


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def manager(tokens, H, blocks=1, scale=2, window=3, total=60, **kw):
    return P.B200KVCacheManager(blocks, 21, tokens, H, 64, device=DEV, num_special_tokens=kw.pop("ns", NS), scale_frames=scale, sliding_window=window,
                                max_total_frames=total, kv_bits=kw.pop("kv_bits", 4), **kw)


def same_rows(got, x, tag):
    """(values, scales) read back are the quantisation of x, bit for bit (signs of zeros too; NaN scales as NaN)."""
    codes, scales = F.quantise(x)
    v, s = got[0].view(torch.uint8).cpu().numpy(), got[1].cpu().numpy()
    want_v = dev(F.values(codes) , torch.float32).to(torch.float8_e4m3fn)
    want_v = torch.where(dev(codes & 8) != 0, -want_v.float().abs(), want_v.float().abs()).to(torch.float8_e4m3fn).view(torch.uint8).cpu().numpy()
    assert (v == want_v).all(), f"{tag}: {int((v != want_v).sum())} of {v.size} values differ"
    want_s = F.SCALES[scales]
    bad = scales == 255
    assert (np.isnan(s) == bad).all() and (s[~bad].astype(np.float64) == want_s[~bad]).all(), f"{tag}: scales differ"


def bound_rows(keys, spread, weighted, out):
    """Few-row kernel, a bf16 result `out` of float64: the final rounding is half a step, 2^-8 |out|.  A logit's error: q, bf16, is exact in half
    precision, products are exact, fp32 sums of at most 128 terms: below (2^-22 + 128 * 2^-24) * sum |q k| / sqrt(D) <= 2^-16 * `spread`; times ln 2 either way
    it moves a weight by that much relatively; exp2 adds 2^-21; fp32 sums over the keys keys * 2^-24 (each addition rounds
    or cuts, relative 2^-23 on partial sums).  Relative weight errors move the result by that share of sum p |v| (`weighted`), twice as numerator and
    denominator both carry them.  A weight is held to 2^-40 of the largest (half of half precision's smallest step, 2^-25, at weights of up to
    2^15): far smaller ones are zero, which moves the result by at most keys * 2^-40 * max|v|, and |v| is below 2^3 in these tests.  In front of V, not
    in the sum that divides, a weight is one half-precision number: half a step is 2^-11 of it, which moves the result by at most 2^-11 `weighted`."""
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -11 + 2 * (2.0 ** -16 * spread + 2.0 ** -21 + keys * 2.0 ** -23)) * weighted + keys * 2.0 ** -37


def spread_of(q, k):
    """The largest sum |q k| / sqrt(D) over (query, key) pairs of any head."""
    return float(np.einsum("nhd,thd->hnt", np.abs(q), np.abs(k)).max()) / np.sqrt(q.shape[-1])


# ---------------------------------------------------------------- what is stored
def special_rows(rs, tokens, H):
    """Rows that quantisation can get wrong among ordinary ones."""
    x = rs.standard_normal((tokens, H, 64)) * np.exp2(rs.randint(-3, 4, (tokens, H, 1)))
    x[0] = 0.0
    x[1] = -0.0
    x[2, :, :16] = np.tile([6, 5, 4, 3.5, 3, 2.5, 2, 1.75, -6, 1.25, 1, 0.75, 0.5, 0.25, -0.25, 0], (H, 1))      # ties at scale 1
    x[3] = rs.standard_normal((H, 64)) * 2.0 ** -17          # around the smallest scales
    x[4] = rs.standard_normal((H, 64)) * 3e4                 # around the largest scale and beyond
    x[5] = 1e38
    x[6, :, 5] = np.nan
    x[7, :, 37] = np.inf
    x[8, :, 63] = -np.inf
    x[9] = 2.0 ** -140                                       # an fp32 subnormal
    x[10, :, 0] = 6 * 1.0625                                 # halfway between two scales
    x[10, :, 16] = 6 * 1.1875
    return x


@pytest.mark.parametrize("patches,H,ns", [(20, 3, 6), (130, 2, 6), (7, 1, 5), (257, 1, 0)])
@pytest.mark.parametrize("kd,vd", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
def test_append_stores_the_quantised_rows(patches, H, ns, kd, vd):
    types = {"f32": torch.float32, "bf16": torch.bfloat16}
    rs = np.random.RandomState(patches + H)
    m = manager(patches + ns, H, ns=ns)
    for t in range(4):
        k, v = special_rows(rs, patches + ns, H).astype(np.float32), special_rows(rs, patches + ns, H).astype(np.float32)
        m.append_frame(0, dev(k, types[kd]), dev(v, types[vd]))
        m.evict_frames(0, 2, 3)
        kv, ks, vv, vs = m.last_frame_fp4(0)
        assert kv.dtype == torch.float8_e4m3fn and tuple(kv.shape) == (patches + ns, H, 64) and ks.dtype == torch.float16 and tuple(ks.shape) == (patches + ns, H, 4)
        same_rows((kv, ks), bf(k), f"frame {t} K")
        same_rows((vv, vs), bf(v), f"frame {t} V")
    # the page itself, byte by byte as the header describes it (patches of the newest frame)
    page = m.scale_patch_pages[0][-1] if len(m.live_window_patch_pages[0]) == 0 else m.live_window_patch_pages[0][-1]
    raw = m.kv_caches[0][page].cpu().numpy()
    for kv, x in ((0, bf(k)), (1, bf(v))):
        for h in range(H):
            codes, scales = F.quantise(x[ns:, h])
            want = F.pack_head(codes, scales, patches)
            assert (raw[kv, h] == want).all()
    assert m.device_status() == 0


def test_every_border_of_every_scale():
    """Blocks of every scale with values on all seven borders between two codes, and on the fp32 numbers on either side of them."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    scales = F.SCALES[1:F.TOP_BYTE + 1]
    blocks = []
    for s in scales:
        for step in (None, 0.0, np.inf):
            x = (borders * s).astype(np.float32)
            if step is not None:
                x = np.nextafter(x, np.float32(step))
            blocks.append(np.concatenate([[6 * s], x, -x, [0.0]]))
    x = np.array(blocks)
    x = np.concatenate([x, np.zeros((-len(x) % 8, 16))]).reshape(-1, 1, 128)
    assert (F.SCALES[F.quantise(x)[1]].reshape(-1)[:3 * len(scales)].reshape(-1, 3) == scales[:, None]).all()
    c = P.DecodeCache(1, 128, DEV, kv_bits=4)
    c.append(dev(x), dev(-x))
    got = c.rows_fp4(0, len(x))
    same_rows(got[:2], x, "K")
    same_rows(got[2:], -x, "V")
    y = x.reshape(-1, 1, 64)                              # the paged cache: the same, rounded to bf16 first
    m = manager(len(y), 1, ns=0)
    m.append_frame(0, dev(y), dev(-y))
    got = m.last_frame_fp4(0)
    same_rows(got[:2], bf(y), "paged K")
    same_rows(got[2:], bf(-y), "paged V")


@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode,norm", [(_lib.ROPE_3D, True), (_lib.ROPE_2D, True), (_lib.ROPE_NONE, False), (_lib.ROPE_3D, False)])
def test_fused_append_is_the_wide_append_quantised(src, mode, norm):
    """qkv with norm and rotation: the 4-bit cache holds the quantisation of exactly what the bf16 cache holds, queries are the same."""
    pph, ppw, H = 9, 15, 3
    T = pph * ppw + NS
    wide, slim = manager(T, H, kv_bits=16), manager(T, H)
    g = torch.Generator(device=DEV).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    params = (1 + 0.1 * rand(64), 0.1 * rand(64), 1 + 0.1 * rand(64), 0.1 * rand(64)) if norm else (None,) * 4
    cs = {_lib.ROPE_3D: P.ops.rope3d_table(4, pph, ppw, NS, DEV), _lib.ROPE_2D: P.ops.rope2d_table(pph, ppw, NS, DEV), _lib.ROPE_NONE: None}[mode]
    for t in range(5):
        buf = rand(T, 3 * H * 64 + 16).to(src)
        qkv = buf[:, :3 * H * 64]                          # rows that do not follow each other
        qa, qb = (x.append_frame_fused(0, qkv, *params, cs, mode) for x in (wide, slim))
        assert torch.equal(qa, qb)
        for x in (wide, slim):
            x.evict_frames(0, 2, 3)
    for a, b in zip(wide._gather_kv(0), slim._gather_kv(0)):
        assert a.shape == b.shape and b.dtype == torch.bfloat16
        assert (host(b) == F.roundtrip(host(a))).all()
    assert slim.device_status() == 0 and wide.build_visible_page_table(0) == slim.build_visible_page_table(0)


def test_a_frame_taken_back_leaves_no_trace():
    rs = np.random.RandomState(3)
    T, H = 30, 2
    m = manager(T, H)
    k = [rs.standard_normal((T, H, 64)) for _ in range(5)]
    for t in range(4):
        m.append_frame(0, dev(k[t]), dev(k[t]))
        m.evict_frames(0, 2, 3)
    before, q = [x.clone() for x in m._gather_kv(0)], dev(k[4], torch.bfloat16)
    out = m.compute_attention(0, q).clone()
    m._defer_eviction = True
    m.append_frame(0, dev(k[4]), dev(k[4]))
    assert not torch.equal(m.compute_attention(0, q), out)
    m.rollback_last_frame(0)
    m._defer_eviction = False
    assert all(torch.equal(a, b) for a, b in zip(before, m._gather_kv(0)))
    assert torch.equal(m.compute_attention(0, q), out)
    m.reset()
    with pytest.raises(_lib.GctError):
        m.last_frame_fp4(0)
    assert float(m.compute_attention(0, q).abs().max()) == 0.0


def test_reading_a_wide_cache_as_fp4_is_refused():
    m = manager(30, 2, kv_bits=16)
    m.append_frame(0, torch.zeros(30, 2, 64, device=DEV), torch.zeros(30, 2, 64, device=DEV))
    with pytest.raises(_lib.GctError):
        m.last_frame_fp4(0)
    lib = _lib.load()
    assert lib.gct_mgr_set_kv_format(m._handle, _lib.KV_FP4, None) == _lib.ERR_INVALID       # bound already
    s = manager(30, 2)
    for page, rows in ((-1, 1), (s.max_num_pages, 1), (0, 25), (0, -1)):
        assert lib.gct_mgr_read_page_fp4(s._handle, 0, page, rows, s.workspace_buffer.data_ptr(), s.workspace_buffer.data_ptr(), None) == _lib.ERR_INVALID


# ---------------------------------------------------------------- attention over the pages
def filled(tokens, H, frames, rs, scale=2, window=3, k_scale=1.0, **kw):
    m = manager(tokens, H, scale=scale, window=window, total=max(frames, 1) + 4, **kw)
    for t in range(frames):
        m.append_frame(0, dev(rs.standard_normal((tokens, H, 64)) * k_scale, torch.bfloat16), dev(rs.standard_normal((tokens, H, 64)), torch.bfloat16))
        m.evict_frames(0, scale, window)
    k, v = (host(x) for x in m._gather_kv(0))
    return m, k, v


@pytest.mark.parametrize("n_q", [1, 2, 6, 8])
@pytest.mark.parametrize("patches,H,frames", [(1, 1, 1), (20, 3, 1), (20, 3, 9), (127, 2, 4), (128, 2, 5), (129, 1, 5), (300, 2, 12), (999, 2, 6)])
def test_few_query_rows(patches, H, frames, n_q):
    T, ns = patches + (NS if patches > 1 else 0), NS if patches > 1 else 0
    if n_q > T:
        pytest.skip("a call has at most a frame's tokens")
    rs = np.random.RandomState(patches + frames)
    m, k, v = filled(T, H, frames, rs, ns=ns)
    q = bf(rs.standard_normal((n_q, H, 64)) * 2)
    want, want_lse, weighted = F.attention(q, k, v)
    tol = bound_rows(len(k), spread_of(q, k), weighted, want)
    for x in (dev(q, torch.bfloat16), dev(q)):
        out, lse = m.compute_attention(0, x, return_lse=True)
        assert out.dtype == torch.bfloat16 and (np.abs(host(out) - want) <= tol).all(), float((np.abs(host(out) - want) / tol).max())
        # the log-sum-exp: a logit error moves it as much; log2 and the sums as above
        assert np.abs(host(lse) - want_lse).max() <= 2.0 ** -16 * spread_of(q, k) + 2.0 ** -21 + len(k) * 2.0 ** -23 + 2.0 ** -22 * np.abs(want_lse).max()
        assert torch.equal(out, m.compute_attention(0, x))
    assert m.device_status() == 0


@pytest.mark.parametrize("scale", [1e-30, 2.0 ** -40, 1.0, 300.0, 2.0 ** 60])
def test_queries_of_any_magnitude(scale):
    """q is brought to the range of half precision by a power of two per row: tiny, ordinary and huge rows side by side."""
    rs = np.random.RandomState(1)
    m, k, v = filled(40, 2, 5, rs)
    q = bf(rs.standard_normal((4, 2, 64)) * np.array([1.0, scale, scale, 0.0])[:, None, None])
    want, _, weighted = F.attention(q, k, v)
    out = host(m.compute_attention(0, dev(q, torch.bfloat16)))
    assert np.isfinite(out).all()
    for i in range(4):                                    # each row by its own spread: a huge one says little, its neighbours as much as ever
        tol = bound_rows(len(k), spread_of(q[i:i + 1], k), weighted[i:i + 1], want[i:i + 1])
        assert (np.abs(out[i:i + 1] - want[i:i + 1]) <= tol).all(), i


@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("scale", [1e-30, 2.0 ** -12, 300.0, 2.0 ** 60])
def test_query_tiles_of_any_magnitude(scale, with_lse):
    """The same through the query tiles, whose CTAs fold scale and reference into the product only where all their rows allow it."""
    rs = np.random.RandomState(2)
    m, k, v = filled(60, 1, 5, rs)
    q = bf(rs.standard_normal((40, 1, 64)) * np.where(np.arange(40) % 7 == 3, scale, np.where(np.arange(40) % 7 == 5, 0.0, 1.0))[:, None, None])
    want, want_lse, weighted = F.attention(q, k, v)
    got = m.compute_attention(0, dev(q, torch.bfloat16), return_lse=with_lse)
    out = host(got[0] if with_lse else got)
    assert np.isfinite(out).all()
    for i in range(40):
        spread = spread_of(q[i:i + 1], k)
        assert (np.abs(out[i] - want[i]) <= bound_frame(len(k), spread, weighted[i], want[i])).all(), i
        if with_lse:
            assert np.abs(host(got[1])[i] - want_lse[i]).max() <= 2.0 ** -16 * spread + 2.0 ** -13 + len(k) * 2.0 ** -23 + 2.0 ** -22 * np.abs(want_lse[i]).max(), i


def test_values_that_are_not_finite_stay_visible_and_hidden_ones_do_not_leak():
    rs = np.random.RandomState(7)
    T, H = 40, 2
    m = manager(T, H, scale=1, window=1, total=40)
    k, v = rs.standard_normal((T, H, 64)), rs.standard_normal((T, H, 64))
    bad = v.copy()
    bad[:, :, :] = np.nan
    # a frame of NaNs, evicted: its page is handed out again, its special rows are behind the last valid ones after a rollback
    m.append_frame(0, dev(k), dev(v))
    m.append_frame(0, dev(bad), dev(bad))
    m.rollback_last_frame(0)
    q = dev(rs.standard_normal((3, H, 64)), torch.bfloat16)
    assert torch.isfinite(m.compute_attention(0, q)).all() and torch.isfinite(m.compute_attention(0, dev(rs.standard_normal((T, H, 64))))).all()
    v[5, 0, 20] = np.inf                                  # one value: its block of sixteen columns of that head
    m.append_frame(0, dev(k), dev(v))
    for rows in (3, T):
        out = host(m.compute_attention(0, dev(rs.standard_normal((rows, H, 64)), torch.bfloat16)))
        assert np.isnan(out[:, 0, 16:32]).all() and np.isfinite(np.delete(out[:, 0], range(16, 32), axis=-1)).all() and np.isfinite(out[:, 1]).all()
    qn = rs.standard_normal((3, H, 64))
    qn[1, 1, 7] = np.nan
    out = host(m.compute_attention(0, dev(qn, torch.bfloat16)))
    assert np.isnan(out[1, 1]).all() and np.isfinite(out[[0, 2], 1]).all()


def test_partial_results_of_page_ranges_merge():
    rs = np.random.RandomState(11)
    m, k, v = filled(150, 2, 9, rs)
    for n_q in (2, 150):
        q = bf(rs.standard_normal((n_q, 2, 64)))
        pages = len(m.build_visible_page_table(0))
        parts, lses = [], []
        for lo, hi in ((0, 2), (2, pages - 1), (pages - 1, pages)):
            m.plan(lo, hi)
            o, l = m.compute_attention_partial(0, dev(q, torch.bfloat16))
            parts.append(o)
            lses.append(l)
        out = host(P.ops.lse_merge(torch.stack(parts), torch.stack(lses)))
        want, _, weighted = F.attention(q, k, v)
        assert (np.abs(out - want) <= bound_frame(len(k), spread_of(q, k), weighted, want)).all()


def test_plans_of_many_pages():
    """More pages than a plan hands over as an argument: 500 frames on pages of seven rows; then few again after a reset."""
    rs = np.random.RandomState(13)
    m, k, v = filled(13, 2, 500, rs, scale=2, window=3)
    assert len(m.build_visible_page_table(0)) > 256
    for n_q in (1, 13):
        q = bf(rs.standard_normal((n_q, 2, 64)))
        want, _, weighted = F.attention(q, k, v)
        for _ in range(2):
            out = host(m.compute_attention(0, dev(q, torch.bfloat16)))
            assert (np.abs(out - want) <= bound_frame(len(k), spread_of(q, k), weighted, want)).all()
    m.reset()
    x = dev(rs.standard_normal((13, 2, 64)), torch.bfloat16)
    m.append_frame(0, x, x)
    k, v = (host(t) for t in m._gather_kv(0))
    want, _, weighted = F.attention(host(x), k, v)
    assert (np.abs(host(m.compute_attention(0, x)) - want) <= bound_frame(len(k), spread_of(host(x), k), weighted, want)).all()
    assert m.device_status() == 0


def bound_frame(keys, spread, weighted, out):
    """Any path: as bound_rows, with weights rounded to half precision (2^-11 relative; below 2^-14 of their scale 2^-25 absolutely) and
    exponentials good to 2^-13 in numerator and denominator, and the merge of ranges in fp32.  Where q is rounded once more with its scale (2^-11 of each
    term of a logit, to either side) nothing is granted for it: the terms cancel."""
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -11 + 2.0 ** -12 + 2 * (2.0 ** -16 * spread + keys * 2.0 ** -23)) * weighted + 2.0 ** -24


@pytest.mark.parametrize("n_q", [9, 16, 17, 64, 128, 129, 256, 257, 1005])
@pytest.mark.parametrize("patches,H,frames", [(20, 3, 9), (128, 2, 5), (129, 1, 5), (300, 2, 12), (999, 2, 6)])
def test_many_query_rows(patches, H, frames, n_q):
    T = patches + NS
    if n_q > T:
        pytest.skip("a call has at most a frame's tokens")
    rs = np.random.RandomState(patches + frames)
    m, k, v = filled(T, H, frames, rs)
    q = bf(rs.standard_normal((n_q, H, 64)) * 2)
    want, want_lse, weighted = F.attention(q, k, v)
    tol = bound_frame(len(k), spread_of(q, k), weighted, want)
    for x in (dev(q, torch.bfloat16), dev(q)):
        out, lse = m.compute_attention(0, x, return_lse=True)
        assert (np.abs(host(out) - want) <= tol).all(), float((np.abs(host(out) - want) / tol).max())
        assert np.abs(host(lse) - want_lse).max() <= 2.0 ** -16 * spread_of(q, k) + 2.0 ** -13 + len(k) * 2.0 ** -23
        assert (np.abs(host(m.compute_attention(0, x)) - want) <= tol).all()
    assert m.device_status() == 0


@pytest.mark.parametrize("patches,n_q", [(122, 128), (300, 306), (300, 40)])
@pytest.mark.parametrize("regime", ["fixed", "off", "too large", "repeated", "some rows repeated"])
def test_softmax_reference(patches, n_q, regime):
    """The fixed reference |q| max|k|, the running maximum it gives way to, and the second pass of a CTA in which a row turned out to lie far
    below its reference: keys that all point against the queries."""
    T, H = patches + NS, 2
    rs = np.random.RandomState(patches)
    m = manager(T, H, scale=1, window=2, total=40)
    against = regime.endswith("repeated")
    u = np.where(rs.standard_normal(64) > 0, 1.0, -1.0)
    for t in range(5):
        k = rs.standard_normal((T, H, 64)) * (0.05 if against else 1.0) - (u if against else 0.0)
        m.append_frame(0, dev(k, torch.bfloat16), dev(rs.standard_normal((T, H, 64)), torch.bfloat16))
        m.evict_frames(0, 1, 2)
    q = rs.standard_normal((n_q, H, 64)) * (8.0 if regime == "too large" else 1.0)
    if against:
        rows = slice(None) if regime == "repeated" else slice(n_q // 2, n_q // 2 + 3)
        q[rows] = 2.2 * u + 0.1 * q[rows]                 # logits of about -18 (26 in base 2), the reference 29
    q = bf(q)
    k, v = (host(x) for x in m._gather_kv(0))
    norms = m.key_norm_max.double().cpu().numpy()[0]
    true_norms = np.sqrt((k ** 2).sum(-1)).max(0)
    assert (norms >= true_norms).all() and (norms <= true_norms * 1.3).all()          # evicted frames had norms of about the same
    reference = np.sqrt((q ** 2).sum(-1)) * norms / 8 * 1.4427
    assert (reference.max() > 30) == (regime == "too large")
    if regime == "off":
        m.set_bounded_mode(False)
    want, want_lse, weighted = F.attention(q, k, v)
    out, lse = m.compute_attention(0, dev(q, torch.bfloat16), return_lse=True)
    tol = bound_frame(len(k), spread_of(q, k), weighted, want)
    assert (np.abs(host(out) - want) <= tol).all(), float((np.abs(host(out) - want) / tol).max())
    assert np.abs(host(lse) - want_lse).max() <= 2.0 ** -16 * spread_of(q, k) + 2.0 ** -13 + len(k) * 2.0 ** -23
    assert m.device_status() == 0
    # the norms found again from the pool alone
    m.rescan_key_norms()
    again = m.key_norm_max.double().cpu().numpy()[0]
    assert (again >= true_norms).all() and (again <= norms * 1.001).all()


# ---------------------------------------------------------------- the camera head's caches
def decode_bound(keys, spread, weighted):
    """fp32 results: as bound_rows without the last rounding, and with q and the weights in two parts (22 bits each: 2^-22 of a logit's terms, 2^-22 of a
    weight); the rounding of the division and of the result, 2^-23, is inside the first terms."""
    return 2 * (2.0 ** -16 * spread + 2.0 ** -20 + keys * 2.0 ** -23) * weighted + 2.0 ** -30


@pytest.mark.parametrize("H,D", [(16, 128), (2, 128), (3, 64), (1, 64)])
@pytest.mark.parametrize("cached,new", [(0, 1), (0, 8), (1, 1), (12, 1), (127, 2), (128, 1), (129, 8), (700, 1), (700, 9), (5, 20), (3, 130), (2001, 8)])
def test_decode_matches_the_definition(H, D, cached, new):
    rs = np.random.RandomState(H * 1000 + D + cached + new)
    c = P.DecodeCache(H, D, DEV, capacity=16, kv_bits=4)
    f32 = lambda a: a.astype(np.float32).astype(np.float64)
    k, v = f32(rs.standard_normal((cached, H, D)) * 1.5), f32(rs.standard_normal((cached, H, D)))
    if cached:
        c.append(dev(k), dev(v))
    q, kn, vn = (f32(rs.standard_normal((new, H, D)) * s) for s in (1.5, 1.5, 1.0))
    kk, vv = F.roundtrip(np.concatenate([k, kn])), F.roundtrip(np.concatenate([v, vn]))
    want, _, weighted = F.attention(q, kk, vv)
    tol = decode_bound(cached + new, spread_of(q, kk), weighted)
    behind = [t.clone() for t in (c.k, c.v)]
    out = c.attend(dev(q), dev(kn), dev(vn), False)
    assert out.dtype == torch.float32 and (np.abs(host(out) - want) <= tol).all(), float((np.abs(host(out) - want) / tol).max())
    assert c.count == cached and all(torch.equal(a, b) for a, b in zip(behind, (c.k, c.v)))      # nothing stored
    out2 = c.attend(dev(q), dev(kn), dev(vn), True)
    assert c.count == cached + new and (np.abs(host(out2) - want) <= tol).all()
    got = c.rows_fp4(0, cached + new)
    same_rows(got[:2], np.concatenate([k, kn]), "K")
    same_rows(got[2:], np.concatenate([v, vn]), "V")
    part = c.rows_fp4(cached, new)
    assert all(torch.equal(a.view(torch.uint8), b[cached:].view(torch.uint8)) for a, b in zip(part, got))
    assert int(c.workspace[:4].view(torch.int32)[0]) == 0


def test_decode_stream_grows_and_is_taken_back():
    H, D = 2, 128
    c = P.DecodeCache(H, D, DEV, capacity=100, kv_bits=4)
    assert c.capacity == 128
    rs = np.random.RandomState(2)
    ks, vs = [], []
    for i, n in enumerate([8] + [1] * 5 + [8] * 40 + [1, 3]):
        q, k, v = (rs.standard_normal((n, H, D)).astype(np.float32) for _ in range(3))
        out = c.attend(dev(q), dev(k), dev(v), True)
        ks.append(k)
        vs.append(v)
    kk, vv = F.roundtrip(np.concatenate(ks)), F.roundtrip(np.concatenate(vs))
    want, _, weighted = F.attention(q.astype(np.float64), kk, vv)
    assert c.count == len(kk) and c.capacity >= c.count and (np.abs(host(out) - want) <= decode_bound(len(kk), spread_of(q, kk), weighted)).all()
    c.truncate(20)
    want, _, weighted = F.attention(q.astype(np.float64), np.concatenate([kk[:20], F.roundtrip(k)]), np.concatenate([vv[:20], F.roundtrip(v)]))
    out = c.attend(dev(q), dev(k), dev(v), False)
    assert (np.abs(host(out) - want) <= decode_bound(23, spread_of(q, kk), weighted)).all()
    for bad in (-1, 21):
        with pytest.raises(ValueError):
            c.truncate(bad)
    for first, rows in ((0, 21), (-1, 2), (5, -1)):
        with pytest.raises(ValueError):
            c.rows_fp4(first, rows)


def test_decode_values_that_are_not_finite():
    H, D = 2, 64
    rs = np.random.RandomState(4)
    c = P.DecodeCache(H, D, DEV, kv_bits=4)
    k, v = rs.standard_normal((40, H, D)), rs.standard_normal((40, H, D))
    v[39, 0, 3] = np.inf
    c.append(dev(k), dev(v))
    c.truncate(39)                                        # the infinite one lies behind the last row
    x = [dev(rs.standard_normal((1, H, D))) for _ in range(3)]
    assert torch.isfinite(c.attend(*x, False)).all()
    c.append(dev(k[39:]), dev(v[39:]))
    out = host(c.attend(*x, False))
    assert np.isnan(out[0, 0, :16]).all() and np.isfinite(out[0, 0, 16:]).all() and np.isfinite(out[0, 1]).all()


def test_decode_refusals():
    c = P.DecodeCache(2, 64, DEV, kv_bits=4)
    t = lambda *s, **k: torch.zeros(*s, device=DEV, **k)
    good = t(1, 2, 64)
    for q, k, v in ((t(1, 2, 128), good, good), (t(1, 3, 64), good, good), (good.bfloat16(), good, good), (good, t(2, 2, 64), good), (good, good, t(2, 2, 64)),
                    (good.cpu(), good, good), (t(2, 64), good, good)):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            c.attend(q, k, v, False)
    with pytest.raises((ValueError, RuntimeError)):
        c.attend(t(0, 2, 64), t(0, 2, 64), t(0, 2, 64), False)
    with pytest.raises(ValueError):
        c.append(t(1, 2, 64), t(1, 2, 32))
    assert c.count == 0
    with pytest.raises(ValueError):
        P.DecodeCache(2, 64, DEV).rows_fp4(0, 0)
    wide = P.DecodeCache(2, 64, DEV, capacity=2)
    wide.append(t(5, 2, 64) + 1, t(5, 2, 64) + 2)
    assert wide.count == 5 and float(wide.k[:5].min()) == 1.0 and float(wide.v[:5].min()) == 2.0


def test_decode_captured_and_replayed():
    """A one-token call that stores nothing is a single launch on fixed addresses: it can be captured; a call in between does not disturb it."""
    H, D = 4, 128
    rs = np.random.RandomState(9)
    c = P.DecodeCache(H, D, DEV, capacity=4096, kv_bits=4)
    c.append(dev(rs.standard_normal((3000, H, D))), dev(rs.standard_normal((3000, H, D))))
    x = [dev(rs.standard_normal((1, H, D))) for _ in range(3)]
    want = c.attend(*x, False).clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = c.attend(*x, False)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(c.attend(*x, False), want)
        torch.cuda.synchronize()


# ---------------------------------------------------------------- together, as a model uses them
def test_stream_of_frames_on_another_stream():
    """Append, eviction, attention and a frame taken back, as a streamed sequence has them, on a stream that is not the default one."""
    pph, ppw, H = 8, 17, 3
    T = pph * ppw + NS
    m = manager(T, H, scale=1, window=2, total=40)
    g = torch.Generator(device=DEV).manual_seed(1)
    w = [1 + 0.1 * torch.randn(64, generator=g, device=DEV) if i % 2 == 0 else 0.1 * torch.randn(64, generator=g, device=DEV) for i in range(4)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for f in range(8):
            qkv = torch.randn(T, 3 * H * 64, generator=g, device=DEV).bfloat16()
            cs = P.ops.rope3d_table(f, pph, ppw, NS, DEV)
            skip = f in (3, 6)
            if skip:
                m._defer_eviction = True
            q = m.append_frame_fused(0, qkv, *w, cs, _lib.ROPE_3D)
            m.evict_frames(0, 1, 2)
            out = m.compute_attention(0, q)
            k, v = (host(x) for x in m._gather_kv(0))
            want, _, weighted = F.attention(host(q), k, v)
            spread = spread_of(host(q), k)
            assert (np.abs(host(out) - want) <= bound_frame(len(k), spread, weighted, want)).all(), f
            one = m.compute_attention(0, q[:1])
            assert (np.abs(host(one) - want[:1]) <= bound_frame(len(k), spread, weighted[:1], want[:1])).all(), f
            if skip:
                m.rollback_last_frame(0)
                m._defer_eviction = False
    assert m.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_stream_on_a_4bit_cache(dtype):
    """Two global blocks through a scale pass, streamed frames and a frame that is no keyframe.  The native layer and the modules fill the cache
    with the same bytes and agree in their outputs; what is cached is the quantisation of what the bf16 cache holds, layer by layer."""
    from test_gpu_blocks import rope3d_pos
    pph, ppw, scale, dim, H = 5, 7, 2, 128, 2
    T = NS + pph * ppw
    torch.manual_seed(3)
    blocks = [P.B200Block(dim=dim, num_heads=H, init_values=0.5, qk_norm=True, rope=object(), kv_cache_sliding_window=2, kv_cache_scale_frames=scale).to(DEV).to(dtype)
              for _ in range(2)]
    make = lambda bits: P.B200KVCacheManager(2, 30, T, H, 64, device=DEV, scale_frames=scale, sliding_window=2, max_total_frames=40, kv_bits=bits)
    xs = [torch.randn(1, scale * T, dim, device=DEV, dtype=dtype)] + [torch.randn(1, T, dim, device=DEV, dtype=dtype) for _ in range(6)]

    def run(mgr, native, one_layer=False):
        outs = []
        for f, x in enumerate(xs):
            frames = scale if f == 0 else 1
            mgr._skip_append = f == 4
            kw = dict(num_patches=T - NS, num_special=NS, enable_3d_rope=True, num_frames=frames, kv_cache=mgr,
                      pos=rope3d_pos(0 if f == 0 else scale + f - 1, frames, pph, ppw, NS))
            with torch.set_grad_enabled(not native), torch.autocast("cuda", dtype=torch.bfloat16):      # gradients on: the modules
                y = x
                for b, blk in enumerate(blocks[:1] if one_layer else blocks):
                    y = blk(y, global_idx=b, **kw)
            outs.append(y.detach())
        return outs

    slim, slim2, wide = make(4), make(4), make(16)
    got, want = run(slim, True), run(slim2, False)
    # the first block's inputs are the same both ways: the same bytes
    assert torch.equal(slim.kv_caches[0], slim2.kv_caches[0]) or dtype == torch.float32
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a.float() - b.float()).abs().max()) <= 3 * 2 ** -7 * float(b.float().abs().max())
    run(wide, True, one_layer=True)
    slim3 = make(4)
    run(slim3, True, one_layer=True)
    for a, b in zip(wide._gather_kv(0), slim3._gather_kv(0)):
        assert (host(b) == F.roundtrip(host(a))).all()
    assert slim.device_status() == slim2.device_status() == 0


def test_many_blocks_and_heads_track_no_key_norms():
    """A geometry whose key norms do not fit the workspace header: every call runs with the running maximum."""
    m = P.B200KVCacheManager(100, 21, 14, 10, 64, device=DEV, scale_frames=1, sliding_window=1, max_total_frames=4, kv_bits=4)
    rs = np.random.RandomState(6)
    k, v, q = (rs.standard_normal((14, 10, 64)) for _ in range(3))
    for b in (0, 99):
        m.append_frame(b, dev(k), dev(v))
        m.append_frame(b, dev(v), dev(k))
    q = bf(q)
    for b in (0, 99):
        kk, vv = (host(x) for x in m._gather_kv(b))
        for n_q in (5, 14):
            want, _, weighted = F.attention(q[:n_q], kk, vv)
            out = host(m.compute_attention(b, dev(q[:n_q], torch.bfloat16)))
            assert (np.abs(out - want) <= bound_frame(len(kk), spread_of(q[:n_q], kk), weighted, want)).all()
    with pytest.raises(RuntimeError):
        m.key_norm_max


def test_attention_captured_into_a_graph():
    """A plan of few pages is a kernel argument: append apart, a whole attention call can be captured and replayed on new queries."""
    rs = np.random.RandomState(8)
    m, k, v = filled(60, 2, 6, rs)
    for n_q in (3, 60):
        q = torch.zeros(n_q, 2, 64, device=DEV, dtype=torch.bfloat16)
        m.compute_attention(0, q)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = m.compute_attention(0, q)
        for seed in range(3):
            x = bf(np.random.RandomState(seed).standard_normal((n_q, 2, 64)))
            q.copy_(dev(x, torch.bfloat16))
            g.replay()
            torch.cuda.synchronize()
            want, _, weighted = F.attention(x, k, v)
            assert (np.abs(host(out) - want) <= bound_frame(len(k), spread_of(x, k), weighted, want)).all()
    assert m.device_status() == 0


@pytest.mark.parametrize("bits", [4, 32])
def test_appends_of_no_rows(bits):
    c = P.DecodeCache(2, 64, DEV, kv_bits=bits)
    none = torch.zeros(0, 2, 64, device=DEV)
    c.append(none, none)
    one = torch.ones(1, 2, 64, device=DEV)
    c.append(one, one)
    c.append(none, none)
    # two equal rows: their mean is what one of them is held as; in 4 bits 1 / 6 rounds to the scale 0.171875, of which it is 5.8 times, held as 6 times
    want = 6 * 0.171875 if bits == 4 else 1.0
    assert c.count == 1 and c.device_status() == 0 and torch.equal(c.attend(one, one, one, False), one * want)


@pytest.mark.parametrize("patches,H,frames,scale,window", [(27, 2, 290, 2, 280), (20, 3, 9, 2, 4), (300, 2, 5, 2, 4)])
def test_query_tiles_of_few_rows_and_many_pages(patches, H, frames, scale, window):
    """Around the number of rows from which on a call takes the tile kernel; the first case has more pages than a plan hands over as an argument."""
    T = patches + NS
    rs = np.random.RandomState(frames)
    m, k, v = filled(T, H, frames, rs, scale=scale, window=window)
    assert (len(m.build_visible_page_table(0)) > 256) == (frames == 290)
    for n_q in (23, 24, 25, 26, T):
        q = bf(rs.standard_normal((n_q, H, 64)) * 2)
        want, want_lse, weighted = F.attention(q, k, v)
        out, lse = m.compute_attention(0, dev(q, torch.bfloat16), return_lse=True)
        tol = bound_frame(len(k), spread_of(q, k), weighted, want)
        assert (np.abs(host(out) - want) <= tol).all()
        assert np.abs(host(lse) - want_lse).max() <= 2.0 ** -16 * spread_of(q, k) + 2.0 ** -13 + len(k) * 2.0 ** -23
        assert (np.abs(host(m.compute_attention(0, dev(q, torch.bfloat16))) - want) <= tol).all()
    assert m.device_status() == 0


def test_exchange_with_one_rank():
    """gct_mgr_attention_exchange with world = 1 takes the partial results of either kernel: one final range of a few rows, several of query tiles."""
    import ctypes as C
    from lingbot_map_b200.cache import _stream_ptr
    lib = _lib.load()
    rs = np.random.RandomState(21)
    m, k, v = filled(306, 2, 9, rs)
    m.plan()
    one = lambda t: (C.c_void_p * 1)(t.data_ptr())
    flags = torch.zeros(64, dtype=torch.int32, device=DEV)
    for epoch, n_q in enumerate((306, 5, 24, 129), 1):
        rb, fb, sl = C.c_size_t(), C.c_size_t(), C.c_int()
        _lib.check(lib.gct_kv_exchange_sizes(n_q, 2, 1, C.byref(rb), C.byref(fb), C.byref(sl)))
        recv = torch.zeros(rb.value // 4, dtype=torch.float32, device=DEV)
        out = torch.zeros(n_q, 2, 64, dtype=torch.bfloat16, device=DEV)
        q = bf(rs.standard_normal((n_q, 2, 64)))
        qd = dev(q, torch.bfloat16)
        _lib.check(lib.gct_mgr_attention_exchange(m._handle, 0, qd.data_ptr(), _lib.BF16, n_q, 0, 1, 1, one(recv), one(out), one(flags), sl.value, epoch,
                                                  _stream_ptr(m.device)))
        want, _, weighted = F.attention(q, k, v)
        assert (np.abs(host(out) - want) <= bound_frame(len(k), spread_of(q, k), weighted, want)).all()
    assert m.device_status() == 0
