"""Rotary positions with several axes and the append to the paged cache, against the plain 64-bit form."""
import pytest
import torch

import paged_oracle as po
from auto_gpu_kernel_b200 import _lib, rotary

FREQ = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)


def make(n, heads=16, axes=1, far=4096, seed=0, pages=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = pages or -(-n // 64) + 2
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=torch.bfloat16)
    pos = torch.randint(0, far + 1, (axes, n), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * 64, generator=gen, device="cuda")[:n].to(torch.int32)
    return dict(q_pe=half(n, heads, 64), ckv=half(n, 512), kpe=half(n, 64), positions=pos, inv_freq=FREQ.float().cuda(),
                pair_axes=[i % axes for i in range(32)], slots=slots, ckv_cache=half(pages, 64, 512),
                kpe_cache=half(pages, 64, 64))


def check(case, interleaved, label="", q_out=None):
    from auto_gpu_kernel_b200 import workspace
    old_ckv, old_kpe = case["ckv_cache"].clone(), case["kpe_cache"].clone()
    q, k = case["q_pe"].double(), case["kpe"].double()
    angle = (case["positions"].double()[case["pair_axes"]] * case["inv_freq"].double()[:, None]).t()
    got = rotary.append(**case, interleaved=interleaved, q_out=q_out)
    assert workspace.check_status() == 0
    want_q = po.rotate(q, angle[:, None], interleaved)
    want_k = po.rotate(k, angle, interleaved)

    def close(got, want, x, what):
        # the bf16 rounding of the result, and of two fp32 products whose sine and cosine are within 2 steps
        a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])
        size = a.abs() + b.abs()
        size = torch.stack((size, size), -1).flatten(-2) if interleaved else torch.cat((size, size), -1)
        bound = 2.0 ** -8 * want.abs() + 6 * 2.0 ** -23 * size
        err = (got.double() - want).abs()
        assert (err <= bound).all(), f"{label}: {what} off by {(err / bound.clamp_min(1e-300)).max():.2f} of its bound"
    close(got, want_q, q, "q")
    stored = case["slots"] >= 0
    to = case["slots"][stored].long()
    close(case["kpe_cache"].view(-1, 64)[to], want_k[stored], k[stored], "k")
    old_ckv.view(-1, 512)[to] = case["ckv"][stored]
    assert torch.equal(case["ckv_cache"].view(torch.int16), old_ckv.view(torch.int16)), label
    rest = torch.ones(old_kpe.numel() // 64, dtype=torch.bool, device="cuda")
    rest[to] = False
    assert torch.equal(case["kpe_cache"].view(-1, 64)[rest].view(torch.int16), old_kpe.view(-1, 64)[rest].view(torch.int16))
    return got


# ------------------------------------------------------------------------------------------ CPU
def test_sections():
    assert rotary.sections(16, 8, 8) == [0] * 16 + [1] * 8 + [2] * 8
    assert rotary.sections(32) == [0] * 32
    for bad in ((16, 8), (33,), (40, -8), ()):
        with pytest.raises(ValueError):
            rotary.sections(*bad)


def test_pair_axes_of_any_sequence():
    import numpy as np
    want = rotary._pack(bytes(rotary.sections(16, 8, 8)), 3)
    axes = rotary.sections(16, 8, 8)
    for form in (axes, tuple(axes), bytes(axes), np.array(axes), np.array(axes, dtype=np.int8), torch.tensor(axes)):
        assert rotary._pack(rotary._axis_bytes(form), 3) == want, type(form)
    for bad in (32, None, [0.0] * 32, np.zeros(32), [-1] * 32, [256] * 32):
        with pytest.raises(ValueError):
            rotary._axis_bytes(bad)
    for bad in (np.zeros(4, dtype=np.int64), np.zeros(64, dtype=np.int8), [0] * 31, [3] * 32, range(0)):
        with pytest.raises(ValueError):                  # (the buffer of four 64-bit numbers has 32 bytes)
            rotary._pack(rotary._axis_bytes(bad), 3)


def test_host_side_argument_errors():
    f = _lib.load().dsa_rotary_append
    ok = dict(q=16, qt=1024, qh=64, c=16, cs=512, k=16, ks=64, p=16, ps=4, axes=2, f=16, pa=0x5555, i=1, s=16, o=16, cc=16, kc=16,
              n=4, h=16, slots=128)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None, None)
    assert call(n=0, q=None) == 0
    for name in ("q", "c", "k", "p", "f", "s", "o", "cc", "kc"):
        assert call(**{name: None}) == -1, name
    for kw in (dict(n=-1), dict(h=0), dict(h=129), dict(axes=0), dict(axes=5), dict(slots=0), dict(ps=-1), dict(cs=511), dict(ks=63),
               dict(qt=63), dict(qh=63), dict(pa=2), dict(pa=3 << 62), dict(axes=1)):
        assert call(**kw) == -2, kw
    for kw in (dict(qt=1028), dict(qh=68), dict(cs=516), dict(ks=68), dict(q=8), dict(c=8), dict(k=8), dict(o=8), dict(cc=8),
               dict(kc=8)):
        assert call(**kw) == -4, kw


def test_plain_rotation_keeps_lengths():
    x = torch.randn(3, 64, dtype=torch.float64)
    for interleaved in (False, True):
        y = po.rotate(x, torch.randn(3, 32, dtype=torch.float64), interleaved)
        assert torch.allclose(y.norm(dim=1), x.norm(dim=1))
        assert torch.equal(po.rotate(x, torch.zeros(3, 32, dtype=torch.float64), interleaved), x)


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,axes", [(1, 16, 1), (1, 1, 3), (2, 5, 2), (17, 16, 3), (63, 17, 4), (64, 128, 1), (300, 33, 3), (5000, 16, 3)])
def test_shapes(n, heads, axes, interleaved):
    check(make(n, heads, axes, seed=n + heads), interleaved, f"{n} x {heads}, {axes} axes")


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_and_negative_positions(interleaved):
    case = make(64, far=2 ** 30, seed=1)
    case["positions"][0, :8] = torch.tensor([0, 1, -1, -131072, 2 ** 31 - 1, -2 ** 31, 1048575, 2 ** 24 + 1], dtype=torch.int32)
    check(case, interleaved, "far")


@pytest.mark.gpu
def test_skipped_strided_and_in_place():
    case = make(100, axes=3, seed=2)
    case["slots"][::7] = -1
    wide = torch.randn(100, 16, 192, device="cuda").to(torch.bfloat16)
    case["q_pe"] = wide[:, :, 128:]                      # the rope part of a wider head
    both = torch.randn(100, 576, device="cuda").to(torch.bfloat16)
    case["ckv"], case["kpe"] = both[:, :512], both[:, 512:]
    case["pair_axes"] = rotary.sections(16, 8, 8)
    keep = wide.clone()
    check(case, False, "strided")
    assert torch.equal(wide, keep)
    plain = make(100, axes=2, seed=3)
    q = plain["q_pe"].clone()
    first = rotary.append(**plain)
    plain["q_pe"] = q
    assert rotary.append(**plain, q_out=q) is q
    assert torch.equal(first, q)


@pytest.mark.gpu
def test_expanded_positions():
    case = make(50, axes=1, seed=8)
    want = rotary.append(**case, interleaved=True)
    case["positions"] = case["positions"].expand(4, -1)          # text: every axis at the same position
    case["pair_axes"] = rotary.sections(8, 8, 8, 8)
    assert torch.equal(check(case, True, "expanded"), want)


@pytest.mark.gpu
def test_bad_slot_is_reported_and_its_query_still_turned():
    from auto_gpu_kernel_b200 import workspace
    case = make(5, seed=4)
    good = rotary.append(**case)
    case["slots"][2] = case["ckv_cache"].shape[0] * 64
    before = case["ckv_cache"].clone()
    got = rotary.append(**case)
    with pytest.raises(RuntimeError, match="outside"):
        workspace.check_status()
    assert torch.equal(got, good) and torch.equal(before.view(torch.int16), case["ckv_cache"].view(torch.int16))


@pytest.mark.gpu
def test_same_rows_as_the_plain_append_at_position_zero():
    from auto_gpu_kernel_b200 import cache_write
    case = make(40, seed=5)
    case["positions"].zero_()
    cc, kc = case["ckv_cache"].clone(), case["kpe_cache"].clone()
    q = rotary.append(**case)
    cache_write.append_kv(case["ckv"], case["kpe"], case["slots"], cc, kc)
    assert torch.equal(q, case["q_pe"])
    assert torch.equal(cc, case["ckv_cache"]) and torch.equal(kc, case["kpe_cache"])


@pytest.mark.gpu
def test_stream_and_graph():
    case = make(33, axes=2, seed=6)
    want = rotary.append(**case)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = rotary.append(**case)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = rotary.append(**case)
    case["positions"].add_(5)
    g.replay()
    fresh = rotary.append(**case)
    torch.cuda.synchronize()
    assert torch.equal(res, fresh) and not torch.equal(res, want)


@pytest.mark.gpu
def test_refusals():
    case = make(8, axes=2, seed=7)

    def refuses(error, **kw):
        with pytest.raises(error):
            rotary.append(**{**case, **kw})
    q = case["q_pe"]
    refuses(ValueError, q_pe=q.float())
    refuses(ValueError, q_pe=q[:, :, :32])
    refuses(ValueError, q_pe=q.repeat(1, 9, 1))
    refuses(ValueError, ckv=case["ckv"][:4])
    refuses(ValueError, kpe=case["kpe"].t())
    refuses(ValueError, positions=case["positions"].long())
    refuses(ValueError, positions=case["positions"].repeat(3, 1))
    refuses(ValueError, positions=case["positions"][:1])            # pairs ask for axis 1
    refuses(ValueError, inv_freq=case["inv_freq"][:31])
    refuses(ValueError, pair_axes=[0] * 31)
    refuses(ValueError, pair_axes=[0] * 31 + [-1])
    refuses(ValueError, pair_axes=32)
    refuses(ValueError, pair_axes=[0] * 31 + [300])
    refuses(ValueError, slots=case["slots"].long())
    refuses(ValueError, kpe_cache=case["kpe_cache"][:1])
    refuses(ValueError, q_out=q[:, :, :32])
    wide = torch.zeros(8, 16, 128, dtype=torch.bfloat16, device="cuda")
    refuses(ValueError, q_pe=wide[:, :, :64], q_out=wide.view(-1)[:8 * 16 * 64].view(8, 16, 64))
    refuses(RuntimeError, q_pe=wide.view(-1)[4:4 + 8 * 16 * 64].view(8, 16, 64))     # not on a 16-byte boundary
    refuses(RuntimeError, slots=case["slots"].cpu())
    refuses(RuntimeError, q_pe=q.cpu())
    empty = {**case, "q_pe": q[:0], "ckv": case["ckv"][:0], "kpe": case["kpe"][:0], "positions": case["positions"][:, :0],
             "slots": case["slots"][:0]}
    assert rotary.append(**empty).shape == (0, 16, 64)


@pytest.mark.gpu
def test_pair_axes_as_an_array():
    import numpy as np
    case = make(20, axes=3, seed=9)
    want = rotary.append(**case)
    case["pair_axes"] = np.array(case["pair_axes"])
    assert torch.equal(rotary.append(**case), want)
    for bad in (np.zeros(4, dtype=np.int64), 32, None):
        with pytest.raises(ValueError, match="pair_axes"):
            rotary.append(**{**case, "pair_axes": bad})
