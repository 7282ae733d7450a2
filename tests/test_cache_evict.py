"""Eviction by accumulated attention weight: the choice against a plain one, the moved rows bit for bit."""
import pytest
import torch

import paged_oracle as po
from auto_gpu_kernel_b200 import _lib

PAGE = 64


def make(lens, budget, seed=0, index=True, wide=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [max(1, -(-max(n, 0) // PAGE)) for n in lens]
    fresh = [max(1, -(-max(0, min(n, budget)) // PAGE)) for n in lens]
    pages = sum(need) + sum(fresh) + 2
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, new = (torch.full((len(lens), max(k) + wide), -1, dtype=torch.int32) for k in (need, fresh))
    at = 0
    for t, counts in ((table, need), (new, fresh)):
        for b, k in enumerate(counts):
            t[b, :k] = perm[at:at + k]
            at += k
    rand = lambda *s: torch.randint(-2 ** 15, 2 ** 15, s, generator=gen, device="cuda", dtype=torch.int16).view(torch.bfloat16)
    ckv, kpe = rand(pages, PAGE, 512), rand(pages, PAGE, 64)
    keys = torch.randint(-128, 128, (pages, PAGE, 1, 132), generator=gen, device="cuda", dtype=torch.int8) if index else None
    weights = torch.rand(len(lens), table.shape[1] * PAGE, generator=gen, device="cuda") ** 4
    return weights, torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda(), new.cuda(), ckv, kpe, keys


def bits(t):
    return t.view(torch.int8 if t.element_size() == 1 else torch.int16)


def check(args, budget, first=0, last=0, label=""):
    from auto_gpu_kernel_b200 import cache_evict, workspace
    weights, lens, table, new, ckv, kpe, keys = args
    old = [t.clone() if t is not None else None for t in (ckv, kpe, keys)]
    got_lens, got_weights, kept = cache_evict.run(weights, lens, table, new, budget, ckv, kpe, keys, first, last)
    assert workspace.check_status() == 0
    want_ckv, want_kpe = old[0].clone().view(-1, 512), old[1].clone().view(-1, 64)
    want_keys = old[2].clone().view(-1, PAGE * 132) if keys is not None else None
    for b, n in enumerate(lens.tolist()):
        n = max(0, min(n, table.shape[1] * PAGE))
        mine = po.evict_choice(weights[b], n, budget, first, last)
        m = len(mine)
        assert int(got_lens[b]) == m == min(n, budget), label
        assert kept[b, :m].tolist() == mine, f"{label}: request {b}"
        assert (kept[b, m:] == -1).all() and (got_weights[b, m:] == 0).all()
        pos = torch.tensor(mine, dtype=torch.long, device="cuda")
        assert torch.equal(got_weights[b, :m].view(torch.int32), weights[b][pos].view(torch.int32))
        if m == 0:
            continue
        src, dst = po.slots_of(table[b], n)[pos], po.slots_of(new[b], m)
        want_ckv[dst], want_kpe[dst] = old[0].view(-1, 512)[src], old[1].view(-1, 64)[src]
        if keys is not None:
            flat = old[2].view(-1, PAGE * 132)
            for width, at in ((128, 0), (4, PAGE * 128)):
                byte = torch.arange(width, device="cuda")
                want_keys[(dst // PAGE)[:, None], at + (dst % PAGE)[:, None] * width + byte] = \
                    flat[(src // PAGE)[:, None], at + (src % PAGE)[:, None] * width + byte]
    # every other row of the caches is as it was
    assert torch.equal(bits(ckv.view(-1, 512)), bits(want_ckv)), f"{label}: ckv"
    assert torch.equal(bits(kpe.view(-1, 64)), bits(want_kpe)), f"{label}: kpe"
    if keys is not None:
        assert torch.equal(keys.view(-1, PAGE * 132), want_keys), f"{label}: index keys"
    return got_lens, got_weights, kept


# ------------------------------------------------------------------------------------------ CPU
def test_host_side_argument_errors():
    f = _lib.load().dsa_cache_evict
    ok = dict(w=16, ws=512, l=16, t=16, ts=8, n=16, ns=4, c=16, k=16, i=None, nl=16, nw=16, nws=200, kept=16, ks=200, b=2, mp=8,
              nmp=4, pages=64, budget=200, first=4, last=64)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None, None)
    assert call(b=0, w=None) == 0
    for name in ("w", "l", "t", "n", "c", "k", "nl", "nw", "kept"):
        assert call(**{name: None}) == -1, name
    for kw in (dict(ws=511), dict(ts=-1), dict(ns=-1), dict(nws=199), dict(ks=199), dict(b=-1), dict(b=65536), dict(mp=0),
               dict(mp=(1 << 24) + 1), dict(nmp=3), dict(pages=0), dict(budget=0), dict(first=-1), dict(last=-1),
               dict(first=137, last=64), dict(pages=(1 << 24) + 1),
               dict(budget=(1 << 30) + 1, nws=1 << 31, ks=1 << 31, nmp=1 << 25)):
        assert call(**kw) == -2, kw
    for name in ("c", "k", "i"):
        assert call(**{name: 8}) == -4, name


def test_plain_choice():
    w = torch.tensor([5.0, 1.0, 1.0, 9.0, 1.0, 0.0, 2.0])
    assert po.evict_choice(w, 7, 4, 1, 1) == [0, 1, 3, 6]           # equal weights: the lower position
    assert po.evict_choice(w, 7, 7, 0, 0) == list(range(7))
    assert po.evict_choice(w, 0, 4, 1, 1) == []
    w[3], w[4] = float("nan"), float("-inf")
    assert po.evict_choice(w, 7, 5, 0, 0) == [0, 1, 2, 5, 6]


def test_cpu_tensors_are_refused():
    from auto_gpu_kernel_b200 import cache_evict
    z = torch.zeros(1, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors required"):
        cache_evict.run(z, z, z, z, 4, z, z)


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (64, 0, 0), (65, 1, 1), (100, 4, 32), (128, 64, 64), (500, 3, 7)])
def test_budgets(budget, first, last):
    check(make([1, 63, 64, 65, 128, 700, 0, 501, 500, 499], budget, seed=budget), budget, first, last, f"budget {budget}")


@pytest.mark.gpu
@pytest.mark.parametrize("lens,budget", [([5000, 4097, 8200], 4096), ([70001], 9000), ([20000, 3, 16384], 2048),
                                         ([140000, 131000], 3000), ([400003], 50), ([9000] * 20, 64),
                                         ([400003], 150), ([9000] * 20, 164)])
def test_long_rows(lens, budget):
    args = make(lens, budget, seed=len(lens), index=len(lens) != 3)
    if budget < 104:                                     # what is always kept does not fit: refused
        with pytest.raises(ValueError, match="keep_first"):
            check(args, budget, 4, 100, str(lens))
        return
    check(args, budget, 4, 100, str(lens))


@pytest.mark.gpu
def test_many_requests():
    lens = torch.randint(0, 400, (600,), generator=torch.Generator().manual_seed(2)).tolist()
    check(make(lens, 150, seed=3, index=False), 150, 2, 20, "600 requests")


@pytest.mark.gpu
def test_ties_zeros_and_odd_values():
    args = make([3000, 3000, 3000, 3000, 3000], 1000, seed=4)
    w = args[0]
    w[0] = 0.0                                           # nothing was ever looked at
    w[1] = (w[1] * 5).floor()                            # mass ties across the border
    w[2, ::3] = float("nan")
    w[2, 1::3] = float("-inf")
    w[3, ::7] = float("inf")
    w[3, 1::7] = -w[3, 1::7]
    w[3, 2::7] = -0.0
    w[3, 3::7] = 0.0
    w[4] = w[4] * 1e-38                                  # down into the subnormals
    # -0 and 0 are one weight for the choice
    check(args, 1000, 10, 10, "ties")
    assert (torch.isnan(args[0]).sum() > 0)


@pytest.mark.gpu
def test_length_beyond_the_table_and_below_zero():
    args = list(make([300, 200], 100, seed=11))
    args[1] = torch.tensor([100000, -3], dtype=torch.int32, device="cuda")
    lens, _, kept = check(args, 100, 3, 10, "cut")
    assert lens.tolist() == [100, 0] and kept[0, -1] == 319       # the table's last position


@pytest.mark.gpu
def test_requests_within_the_budget_may_keep_their_pages():
    args = list(make([100, 900, 64], 300, seed=5))
    for b in (0, 2):
        args[3][b, :2] = args[2][b, :2]
    check(args, 300, 0, 0, "kept pages")


@pytest.mark.gpu
def test_shared_pages_and_strides():
    args = list(make([900, 900], 300, seed=6, wide=3))
    args[2] = args[2][:1].expand(2, -1)                  # both requests read one prefix
    big = torch.zeros(2, args[0].shape[1] + 10, device="cuda")
    big[:, :args[0].shape[1]] = args[0]
    args[0] = big[:, :args[0].shape[1]]
    check(args, 300, 5, 5, "shared")


@pytest.mark.gpu
def test_outputs_wider_than_the_budget_keep_their_other_columns():
    from auto_gpu_kernel_b200 import cache_evict
    w, lens, table, new, ckv, kpe, keys = make([500, 20], 90, seed=7)
    nl = torch.full((2,), 77, dtype=torch.int32, device="cuda")
    nw, kept = torch.full((2, 100), 5.0, device="cuda"), torch.full((2, 100), 55, dtype=torch.int32, device="cuda")
    cache_evict.kernel(w, lens, table, new, 90, ckv, kpe, keys, nl, nw, kept)
    assert nl.tolist() == [90, 20]
    assert (nw[:, 90:] == 5.0).all() and (kept[:, 90:] == 55).all() and (kept[1, 20:90] == -1).all()


@pytest.mark.gpu
def test_bad_pages_are_skipped_and_reported():
    from auto_gpu_kernel_b200 import cache_evict, workspace
    w, lens, table, new, ckv, kpe, keys = make([400, 400], 100, seed=8)
    table[0, 1], new[1, 0] = 1 << 22, -1
    old, old_table = ckv.clone(), table.clone()
    _, _, kept = cache_evict.run(w, lens, table, new, 100, ckv, kpe, keys)
    with pytest.raises(RuntimeError, match="block_table entry outside"):
        workspace.check_status()
    assert kept[0].tolist() == po.evict_choice(w[0], 400, 100, 0, 0)
    for b in (0, 1):
        for j, pos in enumerate(kept[b].tolist()):
            p, q = int(old_table[b, pos // PAGE]), int(new[b, j // PAGE])
            if 0 <= q < ckv.shape[0]:
                want = old[p, pos % PAGE] if p < ckv.shape[0] else old[q, j % PAGE]
                assert torch.equal(bits(ckv[q, j % PAGE]), bits(want))


@pytest.mark.gpu
def test_streams_and_graph():
    from auto_gpu_kernel_b200 import cache_evict, workspace
    args = make([3000, 40, 5000], 700, seed=9)
    want = cache_evict.run(*args[:4], 700, *args[4:], 4, 64)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cache_evict.run(*args[:4], 700, *args[4:], 4, 64)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = cache_evict.run(*args[:4], 700, *args[4:], 4, 64)
    args[0].copy_(torch.rand_like(args[0]))
    args[1].copy_(torch.tensor([2000, 900, 10], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="block_table entry outside"):    # request 1 was given one page
        workspace.check_status()
    for b, n in enumerate((2000, 900, 10)):
        mine = po.evict_choice(args[0][b], n, 700, 4, 64)
        assert res[2][b, :len(mine)].tolist() == mine


@pytest.mark.gpu
@pytest.mark.parametrize("lens,budget", [([3000, 40, 5000], 700), ([90000, 20000], 9000)])
def test_moved_rows_on_another_stream_and_in_a_replay(lens, budget):
    """The rows themselves, from pages that held something else before each run."""
    from auto_gpu_kernel_b200 import cache_evict, workspace
    weights, seq_lens, table, _, ckv, kpe, keys = make([max(lens)] * len(lens), budget, seed=12)
    seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    per = -(-budget // PAGE)
    used = torch.zeros(ckv.shape[0], dtype=torch.bool)
    used[table.cpu().long().flatten()] = True
    new = (~used).nonzero().flatten()[:per * len(lens)].view(len(lens), per).to(torch.int32).cuda()
    caches = (ckv.view(-1, 512), kpe.view(-1, 64), keys.view(-1, PAGE * 132))

    def forget():
        caches[0].view(-1, PAGE, 512)[new.long()] = -1.25
        caches[1].view(-1, PAGE, 64)[new.long()] = 3.5
        caches[2][new.long()] = 77

    def expect(lens):
        """What the caches hold after a move, from the plain choice and the old pages."""
        want = [c.clone() for c in caches]
        for b, n in enumerate(lens):
            mine = torch.tensor(po.evict_choice(weights[b], n, budget, 4, 64), device="cuda")
            src, dst = po.slots_of(table[b], n)[mine], po.slots_of(new[b], len(mine))
            want[0][dst], want[1][dst] = caches[0][src], caches[1][src]
            for width, at in ((128, 0), (4, PAGE * 128)):
                byte = torch.arange(width, device="cuda")
                want[2][(dst // PAGE)[:, None], at + (dst % PAGE)[:, None] * width + byte] = \
                    caches[2][(src // PAGE)[:, None], at + (src % PAGE)[:, None] * width + byte]
        return want

    def same(want, label):
        for name, got, w in zip(("ckv", "kpe", "index keys"), caches, want):
            assert torch.equal(bits(got), bits(w)), f"{label}: {name}"

    def call():
        return cache_evict.run(weights, seq_lens, table, new, budget, ckv, kpe, keys, 4, 64)
    call()
    torch.cuda.synchronize()
    forget()
    want = expect(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    same(want, "another stream")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = call()
    for shorter in (lens, [n - 17 for n in lens], lens[::-1]):
        forget()
        weights.copy_(torch.rand_like(weights))
        seq_lens.copy_(torch.tensor(shorter, dtype=torch.int32))
        want = expect(shorter)
        g.replay()
        torch.cuda.synchronize()
        same(want, f"replay with {shorter}")
        assert res[0].tolist() == [min(n, budget) for n in shorter]
    assert workspace.check_status() == 0


@pytest.mark.gpu
def test_refusals():
    from auto_gpu_kernel_b200 import cache_evict
    w, lens, table, new, ckv, kpe, keys = make([400, 300], 100, seed=10)

    def refuses(error, *a, **kw):
        with pytest.raises(error):
            cache_evict.run(*a, **kw)
    refuses(ValueError, w, lens, table, new, 0, ckv, kpe, keys)
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe, keys, 60, 50)
    refuses(ValueError, w, lens, table, new, 2 ** 30 + 1, ckv, kpe, keys)
    refuses(ValueError, w, lens, table, new, 2 ** 32 + 100, ckv, kpe, keys)
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe, keys, -1, 0)
    refuses(ValueError, w, lens, table, new, 200, ckv, kpe, keys)                 # two new pages hold 128 tokens
    refuses(ValueError, w[:, :300], lens, table, new, 100, ckv, kpe, keys)
    refuses(ValueError, w.double(), lens, table, new, 100, ckv, kpe, keys)
    refuses(ValueError, w, lens.long(), table, new, 100, ckv, kpe, keys)
    refuses(ValueError, w, lens, table, new[:1], 100, ckv, kpe, keys)
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe[:-1], keys)
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe, keys[:-1])
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe, keys, new_token_weights=w)
    refuses(ValueError, w, lens, table, new, 100, ckv, kpe, keys, new_seq_lens=lens)
    refuses(RuntimeError, w, lens.cpu(), table, new, 100, ckv, kpe, keys)
    refuses(RuntimeError, w, lens, table, new, 100, ckv, kpe, keys.cpu())
