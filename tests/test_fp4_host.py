"""The 4-bit caches without a GPU: known answers of the format, sizes, and every refusal that the host makes."""
import ctypes as C

import numpy as np
import pytest
import torch

import lingbot_map_b200 as P
from lingbot_map_b200 import _lib
from oracle import fp4_oracle as F


def test_known_answers_of_the_format():
    x = np.zeros((9, 16))
    x[0, :8] = [6, 5, 4, 3.5, 3, 2.5, 2, 1.75]            # scale 1: ties go to the value with the even number
    x[0, 8:] = [-6, 1.25, 1, 0.75, 0.5, 0.25, -0.25, 0]
    x[1, 0] = 6 * 1.0625                                   # halfway between the scales 1 and 1.125: the even one
    x[2, 0] = 6 * 1.1875                                   # between 1.125 and 1.25: the even one is 1.25
    x[3, 0] = 1e30                                         # beyond the largest scale: saturates at 6 * 10240
    x[4, 0], x[4, 1] = 3 * 2.0 ** -17, 2.0 ** -18          # half the smallest scale: rounds to zero
    x[5, 0] = 6 * 2.0 ** -17                               # the smallest scale
    x[6, 3] = np.nan
    x[7, 3] = np.inf
    codes, scales = F.quantise(x)
    assert codes[0].tolist() == [7, 6, 6, 6, 5, 4, 4, 4, 15, 2, 2, 2, 1, 0, 8, 0]
    assert F.SCALES[scales[:6, 0]].tolist() == [1.0, 1.0, 1.25, 10240.0, 0.0, 2.0 ** -17]
    assert F.dequantise(codes, scales)[3, 0] == 61440.0 and not F.dequantise(codes, scales)[4].any()
    assert scales[6, 0] == scales[7, 0] == 255 and np.isnan(F.dequantise(codes, scales)[6:8]).all()
    assert scales[8, 0] == 0 and not codes[8].any()


def test_every_product_is_a_half_precision_and_a_bf16_number():
    products = np.outer(F.SCALES[:F.TOP_BYTE + 1], F.VALUES)
    assert (products.astype(np.float16).astype(np.float64) == products).all()
    assert (torch.from_numpy(products).to(torch.bfloat16).double().numpy() == products).all()


def test_quotients_in_single_precision_round_as_exact_ones():
    """x / 6 and x / s rounded to fp32 never land on a border that x itself does not lie on: all borders, and the fp32 numbers around them."""
    borders = [(a + b) / 2 for a, b in zip(F.VALUES, F.VALUES[1:])]
    for s in F.SCALES[1:F.TOP_BYTE + 1]:
        for b in borders:
            for x in (np.nextafter(np.float32(b * s), np.float32(0)), np.nextafter(np.float32(b * s), np.float32(np.inf))):
                assert (np.float32(x / np.float32(s)) > b) == (float(x) > b * s) and np.float32(x / np.float32(s)) != b
    for lo, hi in zip(F.SCALES[:F.TOP_BYTE], F.SCALES[1:F.TOP_BYTE + 1]):
        mid = (lo + hi) / 2
        for x in (np.nextafter(np.float32(6 * mid), np.float32(0)), np.nextafter(np.float32(6 * mid), np.float32(np.inf))):
            assert np.float32(x / np.float32(6)) != mid and (np.float32(x / np.float32(6)) > mid) == (float(x) > 6 * mid)


@pytest.mark.parametrize("patches,head_bytes", [(999, 36000), (128, 4608), (129, 4608 + 144), (20, 720), (1, 144), (7, 288)])
def test_pool_size(patches, head_bytes):
    geo = []
    for bits in (16, 4):
        lib, h, g = _lib.load(), C.c_void_p(), _lib.MgrGeometry()
        cfg = _lib.MgrConfig(1, patches + 1, 3, 64, 1, 1, 2, 40)
        _lib.check(lib.gct_mgr_create(C.byref(h), C.byref(cfg), C.byref(g)))
        if bits == 4:
            _lib.check(lib.gct_mgr_set_kv_format(h, _lib.KV_FP4, C.byref(g)))
        geo.append((g.page_size, g.max_patch_pages, g.max_num_pages, g.pool_bytes))
        lib.gct_mgr_destroy(h)
    assert geo[0][:3] == geo[1][:3] and geo[1][3] == geo[1][2] * 2 * 3 * head_bytes
    codes = np.zeros((patches, 64), np.uint8)
    assert F.pack_head(codes, codes[:, :4], patches).size == head_bytes


def test_decode_sizes():
    cache, work = C.c_size_t(), C.c_size_t()
    for heads, dim, capacity in ((16, 128, 1024), (3, 64, 128)):
        _lib.check(_lib.load().gct_decode_fp4_sizes(heads, dim, capacity, C.byref(cache), C.byref(work)))
        assert cache.value == heads * capacity * (dim // 2 + dim // 16) and work.value > 0
    for heads, dim, capacity in ((0, 64, 128), (2, 96, 128), (2, 64, 0), (2, 64, 100)):
        assert _lib.load().gct_decode_fp4_sizes(heads, dim, capacity, C.byref(cache), C.byref(work)) == _lib.ERR_INVALID


def test_unknown_widths_are_refused():
    kw = dict(num_blocks=1, max_num_frames=21, tokens_per_frame=26, num_heads=2, head_dim=64, bookkeeping_only=True)
    for bits in (8, 32, 0, None, "4"):
        with pytest.raises(ValueError):
            P.B200KVCacheManager(kv_bits=bits, **kw)
    with pytest.raises(ValueError):
        P.DecodeCache(2, 64, "cuda", kv_bits=16)
    with pytest.raises(ValueError):
        P.select.install(kv_bits=8)


def test_environment_selects_the_width(monkeypatch):
    for name, wide in (("LINGBOT_B200_KV_BITS", 16), ("LINGBOT_B200_CAMERA_KV_BITS", 32)):
        monkeypatch.delenv(name, raising=False)
        assert P.select._bits_from_env(name, wide) == wide
        monkeypatch.setenv(name, "4")
        assert P.select._bits_from_env(name, wide) == 4
        monkeypatch.setenv(name, "8")
        with pytest.raises(ValueError):
            P.select._bits_from_env(name, wide)


def test_selector_passes_the_width_on():
    made = []
    sel = P.select._manager_selector(type("Ref", (), {}), lambda *a, **k: made.append(k) or "b200", 4)
    assert sel(num_heads=2) == "b200" and made == [dict(num_heads=2, kv_bits=4)]
    sel = P.select._manager_selector(type("Ref", (), {}), lambda *a, **k: made.append(k) or "b200")
    sel(num_heads=2)
    assert made[-1] == dict(num_heads=2)


def test_bookkeeping_is_that_of_the_wide_cache_and_reading_needs_frames():
    kw = dict(num_blocks=1, max_num_frames=21, tokens_per_frame=26, num_heads=2, head_dim=64, bookkeeping_only=True, scale_frames=2, sliding_window=3,
              max_total_frames=40)
    a, b = P.B200KVCacheManager(**kw), P.B200KVCacheManager(kv_bits=4, **kw)
    assert b.kv_bits == 4 and a.kv_bits == 16
    for t in range(9):
        for m in (a, b):
            m.append_frame_bookkeeping(0)
            m.evict_frames(0, 2, 3)
        assert a.build_visible_page_table(0) == b.build_visible_page_table(0) and a.compute_last_page_len(0) == b.compute_last_page_len(0)
    with pytest.raises(RuntimeError):
        b.last_frame_fp4(0)


def test_c_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    h, g = C.c_void_p(), _lib.MgrGeometry()
    cfg = _lib.MgrConfig(1, 26, 2, 64, 6, 2, 3, 40)
    _lib.check(lib.gct_mgr_create(C.byref(h), C.byref(cfg), C.byref(g)))
    assert lib.gct_mgr_set_kv_format(h, 2, None) == _lib.ERR_INVALID and lib.gct_mgr_set_kv_format(None, 1, None) == _lib.ERR_INVALID
    assert lib.gct_mgr_set_kv_format(h, _lib.KV_FP4, None) == _lib.GCT_OK
    assert lib.gct_mgr_read_frame_fp4(h, 0, None, None, None, None, None) == _lib.ERR_INVALID        # nothing bound
    assert lib.gct_mgr_read_page_fp4(h, 0, 0, 1, None, None, None) == _lib.ERR_INVALID
    lib.gct_mgr_destroy(h)
    one = 4096                                             # an address that is never followed: the arguments are refused first
    att = lambda n, cached, cap, D=64, ws=1 << 22, q=one: lib.gct_decode_attention_fp4(q, one, one, n, one, one, cached, cap, 1, 2, D, one, one, ws, None)
    assert att(0, 0, 128) == _lib.ERR_INVALID and att(1, -1, 128) == _lib.ERR_INVALID and att(1, 0, 100) == _lib.ERR_INVALID
    assert att(1, 0, 128, D=32) == _lib.ERR_INVALID and att(1, 0, 128, ws=16) == _lib.ERR_CAPACITY
    assert att(1, 128, 128) == _lib.ERR_CAPACITY and att(3, 126, 128) == _lib.ERR_CAPACITY and att(1, 0, 128, q=one + 4) == _lib.ERR_INVALID
    app = lambda rows, first, cap: lib.gct_decode_append_fp4(one, one, rows, one, one, first, cap, 2, 64, None)
    assert app(-1, 0, 128) == _lib.ERR_INVALID and app(1, -1, 128) == _lib.ERR_INVALID and app(2, 127, 128) == _lib.ERR_CAPACITY
    assert app(0, 128, 128) == _lib.GCT_OK
    read = lambda first, rows, cap: lib.gct_decode_read_fp4(one, one, first, rows, cap, 2, 64, one, one, one, one, None)
    assert read(-1, 1, 128) == _lib.ERR_INVALID and read(0, 129, 128) == _lib.ERR_INVALID and read(120, 9, 128) == _lib.ERR_INVALID
    assert read(128, 0, 128) == _lib.GCT_OK


def test_camera_head_conversion_keeps_the_width():
    """convert_camera_head marks the layers; the caches are made with the first token that they see."""
    from lingbot_map_b200.camera import convert_camera_head

    class Attn(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.qkv, self.gate_proj = torch.nn.Linear(2, 2), None

    head = torch.nn.Module()
    head.trunk = torch.nn.ModuleList([torch.nn.Module() for _ in range(3)])
    for blk in head.trunk:
        blk.attn = Attn()
    assert convert_camera_head(head, 4) == 3 and all(b.attn.b200_kv_bits == 4 for b in head.trunk)
    assert convert_camera_head(head) == 0                   # converted already
    with pytest.raises(ValueError):
        convert_camera_head(head, 8)


def test_converted_camera_heads_take_a_new_width():
    from lingbot_map_b200.camera import convert_camera_head

    class Attn(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.qkv, self.gate_proj = torch.nn.Linear(2, 2), None

    head, blk = torch.nn.Module(), torch.nn.Module()
    blk.attn = Attn()
    head.trunk = torch.nn.ModuleList([blk])
    assert convert_camera_head(head) == 1 and blk.attn.b200_kv_bits == 32
    assert convert_camera_head(head, 4) == 0 and blk.attn.b200_kv_bits == 4


def test_appends_of_no_rows_and_of_other_types():
    lib = _lib.load()
    one = 4096
    assert lib.gct_decode_append_fp4(None, None, 0, one, one, 5, 128, 2, 64, None) == _lib.GCT_OK
    assert lib.gct_decode_append_fp4(None, one, 1, one, one, 5, 128, 2, 64, None) == _lib.ERR_INVALID
    for bits in (4, 32):
        c = P.DecodeCache(2, 64, "cpu", capacity=128, kv_bits=bits)
        with pytest.raises(ValueError):
            c.append(torch.zeros(1, 2, 64, dtype=torch.float64), torch.zeros(1, 2, 64))
        assert c.count == 0 and c.device_status() == 0
