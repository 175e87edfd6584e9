"""What the windowed attention, the rotation and the paged cache refuse, and their C entry
points' checks, without a device."""
from __future__ import annotations

import ctypes

import pytest
import torch

from reversability_amd import _hip, attention, cache, paths


def test_operators_need_a_gpu():
    qkv = torch.zeros(1, 4, 96, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        attention.window_attention(qkv, 1, 2)
    with pytest.raises(ValueError, match="CUDA"):
        attention.rotate_qkv(qkv, 1, attention.Rotary(32, 4, device="cpu"))
    pages = torch.zeros(2, 1, 16, 32, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        cache.append_kv(qkv[0], 1, pages, pages.clone(), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        cache.cached_attention(qkv[0, :, :32].unsqueeze(1), pages, pages.clone(),
                               ints.view(1, 2), ints[:1], ints, 1)
    with pytest.raises(ValueError, match="CUDA"):
        cache.cache_plan(ints.view(1, 2), ints[:1], ints, 4, 16)


@pytest.mark.parametrize("args", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1)])
def test_windows_are_checked(args):
    with pytest.raises(ValueError):
        attention.check_window(args["window"], args.get("sinks", 0), "here")


def test_packed_heads_are_checked():
    qkv = torch.zeros(1, 4, 96, dtype=torch.float16)
    for heads, kv in ((3, 2), (0, None), (1, 0), (-1, None)):
        with pytest.raises(ValueError, match="multiple of kv_heads"):
            attention.packed_heads(qkv, heads, kv, "here")


def test_rotary():
    for bad in (dict(head_dim=48, positions=4), dict(head_dim=64, positions=0),
                dict(head_dim=64, positions=4, base=0.0),
                dict(head_dim=64, positions=4, base=float("nan"))):
        with pytest.raises(ValueError):
            attention.Rotary(device="cpu", **bad)
    rotary = attention.Rotary(32, 70_000, base=500.0, device="cpu")
    angle = 69_999 * 500.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert torch.equal(rotary.table[-1, :, 0], angle.cos().float())
    assert torch.equal(rotary.table[-1, :, 1], angle.sin().float())
    copy = rotary.to("cpu")
    assert copy is not rotary and copy.interleaved == rotary.interleaved
    with pytest.raises(ValueError):
        rotary.check(torch.zeros(1), 64, "here")


def _model(method="baseline"):
    from reversability_amd import build_model
    config = {"model": {"vocab_size": 31, "max_sequence_length": 40, "n_layers": 2, "n_heads": 2,
                        "d_model": 64, "d_ff": 64}, "method": method}
    torch.manual_seed(1)
    return build_model(config)


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_model_with_a_window_on_the_cpu(interleaved):
    """The torch path of enable_attention(window=, sinks=, rotary=): a token's logits depend on
    the tokens it sees through the layers, and on no other."""
    model = _model()
    rotary = attention.Rotary(32, 40, interleaved=interleaved, device="cpu")
    attention.enable_attention(model, window=3, sinks=1, rotary=rotary)
    ids = torch.randint(0, 31, (1, 30))
    changed = ids.clone()
    changed[0, 10] = (changed[0, 10] + 1) % 31
    with torch.no_grad():
        a, b = model(ids)[0], model(changed)[0]
    differs = (a != b).any(1).nonzero()[:, 0].tolist()
    # token 10 reaches two tokens further in each of the two layers
    assert differs and min(differs) == 10 and max(differs) <= 14
    changed = ids.clone()
    changed[0, 0] = (changed[0, 0] + 1) % 31
    with torch.no_grad():
        assert (model(changed)[0] != a).any(1).all()  # the sink: all see it
    with pytest.raises(paths.UnsupportedPathError), paths.strict():
        model(ids)
    with pytest.raises(ValueError, match="Rotary"):
        attention.enable_attention(_model(), rotary=attention.Rotary(64, 40, device="cpu"))
    with pytest.raises(ValueError):
        attention.enable_attention(_model(), window=0)
    attention.enable_attention(model, rotary=attention.Rotary(32, 20, device="cpu"))
    with pytest.raises(ValueError, match="positions of the Rotary table"):
        model(ids)


def test_torch_rotation_is_the_formula():
    qkv = torch.randn(2, 7, 3 * 64, dtype=torch.float64)
    for interleaved in (False, True):
        rotary = attention.Rotary(32, 9, base=50.0, interleaved=interleaved, device="cpu")
        got = attention.reference_rotation(qkv, 2, rotary).view(2, 7, 3, 2, 32)
        x = qkv.view(2, 7, 3, 2, 32)
        assert torch.equal(got[:, :, 2], x[:, :, 2])
        for t in range(7):
            for i in range(16):
                angle = torch.tensor(t * 50.0 ** (-i / 16), dtype=torch.float64)
                c, s = angle.cos().float().double(), angle.sin().float().double()
                j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + 16)
                a, b = x[:, t, :2, :, j], x[:, t, :2, :, k]
                assert torch.allclose(got[:, t, :2, :, j], a * c - b * s, atol=1e-14)
                assert torch.allclose(got[:, t, :2, :, k], a * s + b * c, atol=1e-14)


def test_cache_refuses():
    for bad in (dict(layers=0), dict(pages=0), dict(page_size=24), dict(page_size=8),
                dict(kv_heads=0), dict(head_dim=48), dict(dtype=torch.float32)):
        args = dict(layers=1, pages=2, page_size=16, kv_heads=1, head_dim=32,
                    dtype=torch.float16, device="cpu")
        with pytest.raises(ValueError):
            cache.PagedCache(**{**args, **bad})
    held = cache.PagedCache.for_model(_model(), 3, 16)
    assert held.keys.shape == (2, 3, 2, 16, 32)
    with pytest.raises(ValueError, match="CUDA"):
        held.move(torch.tensor([0, 17]), torch.tensor([17, 3]))
    with pytest.raises(ValueError):
        held.move(torch.tensor([0]), torch.tensor([0, 1]))


def test_decode_refuses():
    model, ids = _model(), torch.zeros(3, dtype=torch.int64)
    held = cache.PagedCache.for_model(model, 3, 16)
    ints = torch.zeros(4, dtype=torch.int32)
    batch = cache.CacheBatch(ints.view(1, 4), ints[:1], ints[:2], 3, 40)
    for bad in ("fp32", "bf16"):
        with pytest.raises(ValueError, match="precision"):
            cache.decode(model, ids, held, batch, precision=bad)
    with pytest.raises(ValueError, match="ids"):
        cache.decode(model, ids.int(), held, batch)
    with pytest.raises(ValueError, match="max_sequence_length"):
        cache.decode(model, ids, held, batch._replace(max_length=41))
    with pytest.raises(ValueError, match="layers"):
        cache.decode(model, ids, cache.PagedCache(1, 3, 16, 2, 32, device="cpu"), batch)
    attention.enable_attention(model, rotary=attention.Rotary(32, 39, device="cpu"))
    with pytest.raises(ValueError, match="Rotary"):
        cache.decode(model, ids, held, batch)


def test_entry_points_validate_without_device():
    lib = _hip.library()
    fake, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    half, f32 = _hip.RV_F16, _hip.RV_F32
    fwd = lambda *a: lib.rv_window_attn_fwd(*a[:-1], None, a[-1], None)
    assert fwd(None, 1, 8, 2, 1, 32, half, 4, 0, fake, fake) == 1
    assert fwd(fake, 1, 0, 2, 1, 32, half, 4, 0, fake, fake) == 2
    assert fwd(fake, 1, 8, 2, 1, 32, half, 0, 0, fake, fake) == 2
    assert fwd(fake, 1, 8, 2, 1, 32, half, 4, -1, fake, fake) == 2
    assert fwd(fake, 1, 8, 3, 2, 32, half, 4, 0, fake, fake) == 3
    assert fwd(fake, 1, 8, 2, 1, 48, half, 4, 0, fake, fake) == 3
    assert fwd(fake, 1, 8, 2, 1, 32, f32, 4, 0, fake, fake) == 3
    assert fwd(odd, 1, 8, 2, 1, 32, half, 4, 0, fake, fake) == 3
    assert fwd(fake, 1, 1 << 40, 2, 1, 32, half, 4, 0, fake, fake) == 3
    need = lib.rv_window_attn_bwd_workspace_bytes(1, 300, 4, 2, 64, 32, 4)
    assert need >= 300 * 4 * 4
    assert lib.rv_window_attn_bwd_workspace_bytes(1, 300, 4, 2, 64, 0, 4) == -2
    assert lib.rv_window_attn_bwd_workspace_bytes(1, 300, 4, 3, 64, 8, 4) == -3
    bwd = lambda ws, n: lib.rv_window_attn_bwd(fake, fake, None, fake, fake, 1, 300, 4, 2, 64, half, 32,
                                               4, fake, ws, n, None)
    assert bwd(None, need) == 4 and bwd(fake, need - 1) == 4 and bwd(odd, need) == 3
    turn = lambda src, tokens, rows, table: lib.rv_rotate_qkv(
        src, fake, tokens, 4, 2, 2, 32, half, table, rows, None, 0, 0, None)
    assert turn(None, 4, 8, fake) == 1 and turn(fake, 4, 8, None) == 1
    assert turn(fake, -1, 8, fake) == 2 and turn(fake, 4, 0, fake) == 2
    assert turn(odd, 4, 8, fake) == 3 and turn(fake, 1 << 40, 8, fake) == 3
    assert turn(fake, 0, 8, fake) == 0
    plan = lambda table, seqs, page, ld=4: lib.rv_cache_plan(
        table, ld, 4, fake, fake, None, seqs, 5, page, fake, fake, None)
    assert plan(None, 1, 16) == 1 and plan(fake, 0, 16) == 2 and plan(fake, 1, 24) == 3
    assert plan(fake, 1, 16, ld=3) == 2
    put = lambda ld=96, q=None, page=16, table=None, pages=3, slots=fake: lib.rv_append_kv(
        fake, ld, q, fake, fake, slots, 4, 1, 1, 32, half, pages, page, table, 8, fake, 0, None)
    assert put(slots=None) == 1 and put(table=fake) == 1 and put(ld=95) == 2 and put(ld=100) == 3
    assert put(page=17) == 3 and put(pages=0) == 2 and put(q=odd) == 3
    see = lambda q=fake, page=16, query=1, tree=None, ld=64, ws=None, n=0, length=64, dtype=half: (
        lib.rv_cached_attn(q, ld, fake, fake, fake, 8, 8, fake, fake, tree, 5, 2, 2, 1, 32, dtype, 9,
                           page, query, length, 0, 0, fake, ws, n, None))
    assert see(q=None) == 1 and see(query=0) == 2 and see(ld=63) == 2 and see(ld=68) == 3
    assert see(page=20) == 3 and see(query=65, tree=fake) == 3 and see(dtype=f32) == 3
    size = lib.rv_cached_attn_workspace_bytes(5, 2, 2, 1, 32, 1, 100_000, 0, 0)
    assert size > 0 and see(length=100_000) == 4
    assert see(length=100_000, ws=fake, n=size - 1) == 4 and see(length=100_000, ws=odd, n=size) == 3
    assert lib.rv_cached_attn_workspace_bytes(5, 2, 3, 2, 32, 1, 64, 0, 0) == -2
    assert lib.rv_cached_attn_workspace_bytes(5, 2, 2, 1, 48, 1, 64, 0, 0) == -3


def test_entry_points_refuse_sizes_whose_products_pass_64_bits():
    lib = _hip.library()
    fake, huge = ctypes.c_void_p(4096), 1 << 62
    names = ("tokens", "seqs", "heads", "kv", "hd", "query", "length", "window", "sinks")
    good = dict(zip(names, (5, 2, 4, 2, 64, 3, 100_000, 7, 4)))
    assert lib.rv_cached_attn_workspace_bytes(*good.values()) >= 0
    for name in names[:4] + names[5:7]:
        assert lib.rv_cached_attn_workspace_bytes(*{**good, name: huge}.values()) < 0, name
    for name in ("window", "sinks"):  # all of what a cache holds
        assert lib.rv_cached_attn_workspace_bytes(*{**good, name: huge}.values()) > 0, name
    sizes = dict(batch=2, seq=300, heads=4, kv=2, hd=64, window=32, sinks=4)
    for name in ("batch", "seq", "heads"):
        args = {**sizes, name: huge}.values()
        assert lib.rv_window_attn_bwd_workspace_bytes(*args) == -3, name
    for name in ("window", "sinks"):
        args = {**sizes, name: huge}.values()
        assert lib.rv_window_attn_bwd_workspace_bytes(*args) > 0, name
    assert lib.rv_cache_plan(fake, 4, 4, fake, fake, None, huge, 5, 16, fake, fake, None) == 3
    assert lib.rv_append_kv(fake, 1 << 30, None, fake, fake, fake, 4, huge, 1, 32, _hip.RV_F16, 3, 16,
                            None, 0, None, 0, None) == 2


def test_partials_of_long_chunks_are_bounded():
    """Chunks that fill the chip by themselves are not cut: partials of every row would be larger
    than the cache."""
    size = _hip.library().rv_cached_attn_workspace_bytes
    assert size(8 * 65536, 8, 32, 8, 128, 65536, 65536, 0, 0) == 0
    for seqs in (1, 4, 32):
        for query in (1, 7, 64, 512, 4096):
            for length in (512, 12000, 1 << 20):
                nbytes = size(seqs * query, seqs, 32, 8, 128, query, length, 0, 0)
                # 2048 blocks of 128 rows and one more for each row, of 130 fp32 values
                most = (2048 * 128 + max(query * 32, 2048 * 128)) * 130 * 4
                assert 0 <= nbytes <= seqs * most, (seqs, query, length, nbytes)


def test_cached_attention_refuses_an_output_in_its_operands():
    """Three tokens of 64 values (384 bytes) and caches of 9216: one byte more on either side of an
    operand is refused, also where the rows of q are strided."""
    lib = _hip.library()
    at = ctypes.c_void_p
    q, keys, values = 1 << 20, 2 << 20, 3 << 20

    def call(out, ld=64):
        return lib.rv_cached_attn(at(q), ld, at(keys), at(values), at(4096), 8, 8, at(4096), at(4096),
                                  None, 3, 2, 2, 1, 32, _hip.RV_F16, 9, 16, 1, 64, 0, 0, at(out),
                                  None, 0, None)
    for first, size in ((q, 384), (keys, 9216), (values, 9216)):
        for out in (first, first - 368, first + size - 16):
            assert call(out) == 3
    assert call(q + 2048 + 112, ld=512) == 3  # (rows at 0, 1024 and 2048 bytes)


def test_partials_of_windows_are_those_of_cut_blocks():
    """The backward's workspace: D and the largest |dO| of 32 queries a head, and fp32 partials of
    the keys' gradients.  At sizes where the keys behind the sinks' fill the chip uncut, only the
    sinks' blocks have them: at most 4096 chunks and one more a block, 128 keys and values each, and
    less than qkv itself."""
    size = _hip.library().rv_window_attn_bwd_workspace_bytes
    for batch, seq, heads, kv, hd, window, sinks in (
            (2, 16384, 10, 10, 128, 2048, 4), (1, 65536, 32, 32, 128, 4096, 4),
            (1, 1 << 20, 16, 16, 128, 2048, 4), (16, 2048, 16, 16, 64, 512, 4),
            (64, 2048, 8, 8, 32, 128, 200)):
        rows = 4 * (batch * heads * seq + 4) + 4 * (batch * heads * (seq // 32 + 1) + 4)
        blocks = batch * kv * -(-sinks // 128)
        most = rows + (4096 + blocks) * 2 * 128 * hd * 4
        nbytes = size(batch, seq, heads, kv, hd, window, sinks)
        assert 0 < nbytes <= most, (seq, nbytes, most)
        assert nbytes < batch * seq * (heads + 2 * kv) * hd * 2  # qkv's
