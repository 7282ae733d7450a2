"""Outputs that share memory with an input or with one another are refused by the operators over the paged caches; column
ranges of one buffer and weights that grow in place are not."""
import math

import pytest
import torch

import paged_oracle as po
from auto_gpu_kernel_b200 import _lib

PAGE = 64
GAP = 1 << 40
SCALE = 1.0 / math.sqrt(192.0)


# ------------------------------------------------------------------------------------------ CPU
def never_launches():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: a call that is not refused would launch")
    return _lib.load()


def pointers(names):
    return {name: (i + 1) * GAP for i, name in enumerate(names)}


def test_attention_refuses_every_pair_on_the_host():
    lib = never_launches()
    p = pointers(["q", "qp", "c", "k", "l", "t", "out", "lse", "w", "nw", "ws"])
    size = lib.dsa_paged_attn_workspace_bytes(2, 1, 16, 8, 1)

    def call(ws=600, nws=700, **at):
        a = {**p, **at}
        return lib.dsa_paged_attn(a["q"], a["qp"], a["c"], a["k"], a["l"], a["t"], 8, 1.0, a["out"], a["lse"], a["w"], ws, a["nw"],
                                  nws, 2, 1, 16, 4, 8, a["ws"], size, None, None)
    bytes_of = dict(q=2 * 16 * 1024, qp=2 * 16 * 128, c=4 * 64 * 1024, k=4 * 64 * 128, l=8, t=64, w=4 * (600 + 512),
                    out=2 * 16 * 1024, lse=2 * 16 * 4, nw=4 * (700 + 512), ws=size)
    for name in ("out", "lse", "nw", "ws"):
        for other, held in bytes_of.items():
            if other == name:
                continue
            assert call(**{name: p[other]}) == -7, (name, other)
            last = p[other] + (held - 1) // 256 * 256                       # the last aligned address inside
            assert call(**{name: last}) == -7, (name, other)
            before = p[other] - (bytes_of[name] - 1) // 256 * 256           # ends inside the other one
            assert call(**{name: before}) == -7, (name, other)
    assert call(w=p["nw"]) == -7                                           # one address, two pitches


def test_eviction_refuses_every_pair_on_the_host():
    lib = never_launches()
    names = ["w", "l", "t", "n", "c", "k", "i", "nl", "nw", "kept"]
    p = pointers(names)

    def call(**at):
        a = {**p, **at}
        return lib.dsa_cache_evict(a["w"], 512, a["l"], a["t"], 8, a["n"], 4, a["c"], a["k"], a["i"], a["nl"], a["nw"], 200, a["kept"],
                                   200, 2, 8, 4, 64, 200, 4, 64, None, None)
    for name in ("c", "k", "i", "nl", "nw", "kept"):
        for other in names:
            if other != name:
                assert call(**{name: p[other]}) == -7, (name, other)


def test_rotary_refuses_every_pair_on_the_host():
    lib = never_launches()
    names = ["q", "c", "k", "p", "f", "s", "o", "cc", "kc"]
    p = pointers(names)

    def call(qt=1024, qh=64, **at):
        a = {**p, **at}
        return lib.dsa_rotary_append(a["q"], qt, qh, a["c"], 512, a["k"], 64, a["p"], 4, 2, a["f"], 0x5555, 1, a["s"], a["o"], a["cc"],
                                     a["kc"], 4, 16, 128, None, None)
    for name, others in (("o", "ckpfs"), ("cc", "qpfs"), ("kc", "qpfs")):
        for other in others:
            assert call(**{name: p[other]}) == -7, (name, other)
    assert call(o=p["cc"]) == -7 and call(o=p["kc"]) == -7 and call(kc=p["cc"]) == -7
    assert call(o=p["q"], qt=2048) == -7 and call(o=p["q"], qt=64, qh=256) == -7     # not the same rows in place
    assert call(o=p["q"] + 1024) == -7


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_attention_refuses_and_allows():
    from test_paged_attention import make
    from auto_gpu_kernel_b200 import paged_attention, workspace
    args = make([300, 70], seed=60)
    q_nope, q_pe, ckv, kpe, lens, table = args
    width = table.shape[1] * PAGE
    out, lse = torch.empty_like(q_nope), torch.empty(2, 16, device="cuda")
    flat = torch.zeros(1 << 16, device="cuda")

    def refuses(**kw):
        with pytest.raises(ValueError, match="overlap"):
            paged_attention.run(*args, SCALE, **kw)
    refuses(output=q_nope)
    refuses(output=ckv.view(-1)[:q_nope.numel()].view(q_nope.shape))
    refuses(lse=q_pe.view(-1).view(torch.float32)[:32].view(2, 16))
    refuses(output=out, lse=out.view(-1).view(torch.float32)[64:96].view(2, 16))
    refuses(new_token_weights=flat[:2 * width].view(2, width), lse=flat[width:width + 32].view(2, 16))
    refuses(new_token_weights=flat[width:3 * width].view(2, width), token_weights=flat[:2 * width].view(2, width))
    refuses(new_token_weights=kpe.view(-1).view(torch.float32)[:2 * width].view(2, width))
    rows = flat[:2 * 2 * width].view(2, 2 * width)
    refuses(token_weights=rows[:, :width], new_token_weights=rows[:, width // 2:width // 2 + width])
    # two column ranges of one buffer are apart
    rows.copy_(torch.rand_like(rows))
    old = rows.clone()
    got, got_lse = paged_attention.run(*args, SCALE, token_weights=rows[:, :width], new_token_weights=rows[:, width:])
    assert workspace.check_status() == 0
    want = po.attend(*args, SCALE, old[:, :width])
    held = torch.arange(width, device="cuda")[None] < lens[:, None]
    po.check_attend(got, got_lse, want, 300, torch.where(held, rows[:, width:], old[:, :width]), old[:, :width], 16, "columns")
    assert torch.equal(rows[:, :width], old[:, :width]) and torch.equal(rows[:, width:][~held], old[:, width:][~held])


@pytest.mark.gpu
def test_eviction_refuses_and_allows():
    from test_cache_evict import make
    from auto_gpu_kernel_b200 import cache_evict, workspace
    w, lens, table, new, ckv, kpe, keys = make([400, 300], 100, seed=61)
    flat = torch.zeros(4096, device="cuda")

    def refuses(**kw):
        with pytest.raises(ValueError, match="overlap"):
            cache_evict.run(w, lens, table, new, 100, ckv, kpe, keys, **kw)
    ints = lambda t: t.view(-1).view(torch.int32)
    refuses(kept_positions=ints(w)[:200].view(2, 100))
    refuses(kept_positions=flat[:200].view(torch.int32).view(2, 100), new_token_weights=flat[100:300].view(2, 100))
    refuses(kept_positions=flat[:200].view(torch.int32).view(2, 100), new_seq_lens=flat[199:201].view(torch.int32))
    refuses(new_seq_lens=lens)
    refuses(new_seq_lens=table.view(-1)[:2])
    refuses(new_seq_lens=new.view(-1)[1:3])
    refuses(new_token_weights=kpe.view(-1).view(torch.float32)[:200].view(2, 100))
    tables = torch.zeros(2, table.shape[1] + 200, dtype=torch.int32, device="cuda")
    tables[:, :table.shape[1]] = table
    with pytest.raises(ValueError, match="overlap"):                        # the choice over the table it is read by
        cache_evict.run(w, lens, tables[:, :table.shape[1]], new, 100, ckv, kpe, keys, kept_positions=tables[:, 4:104])
    # columns of one buffer: the weights in front, the kept ones behind them
    width = w.shape[1]
    both = torch.zeros(2, width + 100, device="cuda")
    both[:, :width] = w
    plain = cache_evict.run(w, lens, table, new, 100, ckv, kpe, keys)
    got = cache_evict.run(both[:, :width], lens, tables[:, :table.shape[1]], new, 100, ckv, kpe, keys,
                          new_token_weights=both[:, width:], kept_positions=tables[:, table.shape[1]:table.shape[1] + 100])
    assert workspace.check_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(plain, got)) and torch.equal(both[:, :width], w)
    assert torch.equal(tables[:, :table.shape[1]], table)


@pytest.mark.gpu
def test_rotary_refuses_and_allows():
    from test_rotary import make
    from auto_gpu_kernel_b200 import rotary, workspace
    case = make(8, axes=2, seed=62)

    def refuses(**kw):
        with pytest.raises(ValueError, match="overlap"):
            rotary.append(**{**case, **kw})
    q = case["q_pe"]
    block = torch.zeros(8, 16, 128, dtype=torch.bfloat16, device="cuda")
    refuses(q_out=case["ckv_cache"].view(-1)[:q.numel()].view(q.shape))
    refuses(q_out=case["kpe_cache"].view(-1)[:q.numel()].view(q.shape))
    rows = torch.zeros(8 * 1024 + 512, dtype=torch.bfloat16, device="cuda")
    refuses(q_out=rows[:8192].view(q.shape), ckv=rows[4096:8192].view(8, 512))
    refuses(q_out=rows[:8192].view(q.shape), kpe=rows[8192 - 512:8192].view(8, 64))
    refuses(q_pe=rows[:8192].view(q.shape), q_out=rows[512:8704].view(q.shape))
    refuses(q_pe=block[:, :, :64], q_out=block.view(-1)[:8192].view(q.shape))
    refuses(kpe_cache=case["ckv_cache"].view(-1)[:case["kpe_cache"].numel()].view_as(case["kpe_cache"]))
    # rows of the caches that are stored again in another place
    case["slots"].copy_(torch.arange(64, 72, dtype=torch.int32))
    case["ckv"], case["kpe"] = case["ckv_cache"].view(-1, 512)[:8], case["kpe_cache"].view(-1, 64)[:8]
    other = {**case, "ckv": case["ckv"].clone(), "kpe": case["kpe"].clone(), "ckv_cache": case["ckv_cache"].clone(),
             "kpe_cache": case["kpe_cache"].clone()}
    assert torch.equal(rotary.append(**case), rotary.append(**other)) and workspace.check_status() == 0
    assert torch.equal(case["ckv_cache"], other["ckv_cache"]) and torch.equal(case["kpe_cache"], other["kpe_cache"])
