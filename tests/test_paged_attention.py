"""Dense attention over the paged cache: against the plain 64-bit form at lengths, head counts and tables where it can
go wrong; refusals; streams and graphs."""
import math

import pytest
import torch

import paged_oracle as po
from auto_gpu_kernel_b200 import _lib

PAGE = 64
SCALE = 1.0 / math.sqrt(192.0)


def make(lens, heads=16, tokens=1, seed=0, spare=2, extra_cols=0, device="cuda"):
    """Shuffled private pages; the rows behind a request's length hold NaN and infinities."""
    gen = torch.Generator(device=device).manual_seed(seed)
    need = [max(0, -(-n // PAGE)) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), max(max(need), 1) + extra_cols), 0, dtype=torch.int32)
    ckv = torch.randn(pages, PAGE, 512, generator=gen, device=device, dtype=torch.bfloat16)
    kpe = torch.randn(pages, PAGE, 64, generator=gen, device=device, dtype=torch.bfloat16)
    at = 0
    for b, (n, k) in enumerate(zip(lens, need)):
        table[b, :k] = perm[at:at + k]
        if k and n % PAGE:
            ckv[perm[at + k - 1], n % PAGE:] = float("nan")
            kpe[perm[at + k - 1], n % PAGE:] = float("inf")
        at += k
    ckv[perm[at:]] = float("nan")
    rows = len(lens) * tokens
    q_nope = torch.randn(rows, heads, 512, generator=gen, device=device, dtype=torch.bfloat16)
    q_pe = torch.randn(rows, heads, 64, generator=gen, device=device, dtype=torch.bfloat16)
    return q_nope, q_pe, ckv, kpe, torch.tensor(lens, dtype=torch.int32, device=device), table.to(device)


def run_and_check(args, label="", weights=False):
    from auto_gpu_kernel_b200 import paged_attention, workspace
    lens, table = args[4], args[5]
    width = table.shape[1] * PAGE
    old = new = None
    if weights:
        gen = torch.Generator(device="cuda").manual_seed(5)
        old = torch.rand(len(lens), width + 3, generator=gen, device="cuda")
        new = torch.full_like(old, -7.0)
    out, lse = paged_attention.run(*args, SCALE, token_weights=old, new_token_weights=new)
    assert workspace.check_status() == 0
    want = po.attend(*args, SCALE, old)
    longest = int(lens.max())
    held = None
    if weights:
        held = torch.arange(width + 3, device="cuda")[None] < lens[:, None]
        assert (new[~held] == -7.0).all(), f"{label}: entries behind the length were written"
        po.check_attend(out, lse, want, longest, torch.where(held, new, old), old, args[0].shape[1], label)
    else:
        po.check_attend(out, lse, want, longest, label=label)
    assert (out[torch.isinf(lse)] == 0).all()
    return out, lse


# ------------------------------------------------------------------------------------------ CPU
def test_host_side_argument_errors():
    lib = _lib.load()
    f = lib.dsa_paged_attn
    big = 1 << 40
    ok = dict(q=16, p=16, c=16, k=16, l=16, t=16, ts=8, sc=1.0, o=16, lse=16, w=None, ws=0, nw=None, nws=0, b=2, n=1, h=16,
              pages=4, mp=8, buf=256, size=big)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None, None)
    assert call(b=0, q=None) == 0
    for name in ("q", "p", "c", "k", "l", "t", "o", "lse", "buf"):
        assert call(**{name: None}) == -1, name
    for kw in (dict(b=-1), dict(b=65536), dict(n=0), dict(h=0), dict(h=129), dict(n=600, h=128), dict(pages=0), dict(mp=0),
               dict(mp=(1 << 24) + 1), dict(pages=(1 << 24) + 1), dict(ts=-1), dict(w=16), dict(nw=16, nws=511),
               dict(nw=16, nws=512, w=16, ws=511)):
        assert call(**kw) == -2, kw
    assert call(size=255) == -3
    for name in ("q", "p", "c", "k", "o", "buf"):
        assert call(**{name: 8 if name != "buf" else 128}) == -4, name


def test_workspace_holds_partials_and_logits():
    lib = _lib.load()
    size = lib.dsa_paged_attn_workspace_bytes
    assert size(0, 1, 16, 8, 0) == 256
    plain, logits = size(64, 1, 16, 512, 0), size(64, 1, 16, 512, 1)
    assert logits - plain == 64 * 512 * 16 * 64 * 4        # fp32 logits of every cached token and query row
    assert plain % 256 == 0
    assert size(1, 1, 16, 64, 0) >= 64 * 2 * 16 * 514 * 4   # a request over 64 CTAs
    assert size(1, 1, 16, 1, 0) == 256                     # whole requests leave no partial results
    assert size(1, 4096, 16, 512, 0) == 256                # nor do more row blocks than SMs


@pytest.mark.parametrize("rows", [16, 64, 128])
def test_requests_are_cut_where_that_was_measured_to_be_faster(rows):
    """The plan shows in the workspace: whole requests leave no partial results.  148 SMs; requests, pages of the table, and
    whether whole ones took less time in the geometric mean over full, evenly and logarithmically spread lengths."""
    size = _lib.load().dsa_paged_attn_workspace_bytes
    measured = {
        16: [(1, 2, True), (1, 8, False), (8, 8, False), (32, 4, True), (32, 8, False), (64, 4, True), (64, 12, False), (100, 12, True),
             (100, 16, False), (148, 16, True), (148, 24, False), (160, 8, True), (160, 12, False), (200, 12, True), (200, 16, False),
             (300, 8, True), (300, 16, True), (300, 24, False), (450, 16, True), (450, 24, True), (700, 16, True), (1000, 12, True)],
        64: [(1, 2, True), (1, 8, False), (8, 8, False), (32, 4, True), (32, 12, False), (64, 4, True), (64, 12, False), (100, 12, True),
             (100, 16, False), (148, 16, True), (148, 24, False), (160, 8, True), (160, 12, False), (200, 12, True), (200, 16, False),
             (300, 16, True), (300, 24, False), (450, 16, True), (450, 24, True), (700, 16, True)],
        128: [(1, 2, True), (1, 8, False), (8, 4, True), (8, 8, False), (32, 8, True), (32, 12, False), (64, 12, True), (64, 24, False),
              (100, 12, True), (100, 16, False), (148, 16, True), (148, 32, False), (160, 16, True), (160, 32, False), (200, 16, True),
              (300, 24, True), (450, 24, True), (700, 16, True)]}
    for batch, pages, whole in measured[rows]:
        assert (size(batch, 1, rows, pages, 0) == -(-8 * batch // 256) * 256) == whole, (batch, pages)


def test_cpu_tensors_are_refused():
    from auto_gpu_kernel_b200 import paged_attention
    args = make([70, 5], device="cpu")
    with pytest.raises(RuntimeError, match="CUDA tensors required"):
        paged_attention.run(*args, SCALE)


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [64], [0], [63, 64, 65, 0, 1, 127, 128, 129], [1000], [5000, 1, 0, 333]])
def test_lengths(lens):
    run_and_check(make(lens), str(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 5, 15, 16, 17, 31, 32, 33, 64, 100, 128])
def test_head_counts(heads):
    run_and_check(make([300, 77, 1, 640], heads=heads, seed=heads), f"{heads} heads", weights=heads in (5, 33, 128))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(2, 16), (3, 16), (4, 16), (5, 5), (8, 16), (70, 1), (130, 3)])
def test_several_new_tokens(tokens, heads):
    # requests shorter than their new tokens: the first of these see nothing
    run_and_check(make([257, 64, 1, 2, 0, 66, 700], heads=heads, tokens=tokens, seed=tokens), f"{tokens} tokens", weights=True)


@pytest.mark.gpu
def test_a_prompt_chunk():
    """More row blocks than SMs: every CTA walks the whole cache."""
    run_and_check(make([1500, 700], tokens=640, seed=40), "640 tokens", weights=True)


@pytest.mark.gpu
def test_many_requests_share_a_cta():
    gen = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 200, (700,), generator=gen).tolist()
    run_and_check(make(lens, seed=2), "700 requests", weights=True)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,most,heads,extra", [(148, 300, 16, 0), (149, 300, 16, 0), (297, 130, 16, 0), (300, 200, 16, 60),
                                                    (500, 64, 5, 0), (1100, 70, 16, 40), (30, 500, 64, 0), (200, 130, 48, 0),
                                                    (160, 150, 33, 50), (75, 200, 100, 0)])
def test_requests_left_whole_and_cut(batch, most, heads, extra):
    """One request per CTA, several per CTA, and (in a table much wider than the lengths) ranges that cut them."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, most + 1, (batch,), generator=gen).tolist()
    lens[0], lens[-1] = most, 0
    run_and_check(make(lens, heads=heads, seed=batch, extra_cols=extra), f"{batch} x {most}, {heads} heads", weights=batch % 2 == 0)


@pytest.mark.gpu
def test_one_long_request_over_all_ctas():
    run_and_check(make([70001], seed=3), "70001 tokens", weights=True)


@pytest.mark.gpu
def test_long_and_short_mixed():
    run_and_check(make([20000, 3, 9000, 64, 0, 12345], seed=4), "mixed", weights=True)
    run_and_check(make([20000, 3, 9000, 64, 0, 12345], heads=32, seed=4), "mixed, 32 heads")


@pytest.mark.gpu
def test_table_wider_than_the_lengths_and_strided():
    args = list(make([100, 300], extra_cols=9, seed=6))
    wide = torch.full((2, args[5].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :args[5].shape[1]] = args[5]
    args[5] = wide[:, :args[5].shape[1]]
    run_and_check(args, "strided table", weights=True)


@pytest.mark.gpu
def test_requests_may_share_pages():
    args = list(make([500], seed=7))
    args[0], args[1] = args[0].repeat(3, 1, 1), args[1].repeat(3, 1, 1)
    args[4] = torch.tensor([500, 129, 500], dtype=torch.int32, device="cuda")
    args[5] = args[5].expand(3, -1)                      # row stride 0
    args[2][torch.isnan(args[2])] = 0.5                  # 129 ends inside a page that others hold
    out, _ = run_and_check(args, "shared", weights=True)
    assert not torch.equal(out[0], out[1])


@pytest.mark.gpu
def test_length_beyond_the_table_is_cut():
    args = list(make([128], seed=8))
    args[4] = torch.tensor([100000], dtype=torch.int32, device="cuda")
    run_and_check(args, "cut")
    args[4] = torch.tensor([-5], dtype=torch.int32, device="cuda")
    from auto_gpu_kernel_b200 import paged_attention
    out, lse = paged_attention.run(*args, SCALE)
    assert (out == 0).all() and torch.isinf(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 1 << 20, -(1 << 31)])
def test_bad_pages_are_left_out_and_reported(bad):
    from auto_gpu_kernel_b200 import paged_attention, workspace
    args = list(make([400, 200, 64], seed=9))
    args[5][0, 2] = bad
    args[5][2, 0] = bad                                  # a request with nothing else
    old = torch.rand(3, args[5].shape[1] * PAGE, device="cuda")
    new = old.clone()
    out, lse = paged_attention.run(*args, SCALE, token_weights=old, new_token_weights=new)
    with pytest.raises(RuntimeError, match="block_table entry outside"):
        workspace.check_status()
    assert (out[2] == 0).all() and torch.isinf(lse[2]).all()
    want = po.attend(*args, SCALE, old)
    po.check_attend(out, lse, want, 400, new, old, 16, "bad page")
    assert torch.equal(new[0, 128:192], old[0, 128:192]) and torch.equal(new[2], old[2])


@pytest.mark.gpu
def test_sharp_rows_and_rising_logits():
    """Logits that rise along the cache refresh the running maximum on every tile; sharp ones leave one weight."""
    args = list(make([1500, 900], seed=10))
    rise = torch.linspace(0.1, 6.0, 1500, device="cuda")
    for b, n in ((0, 1500), (1, 900)):
        slot = po.slots_of(args[5][b], n)
        args[2].view(-1, 512)[slot] = args[0][b, 0].float().mul(rise[:n, None]).to(torch.bfloat16)
    run_and_check(args, "rising", weights=True)
    args[0] = args[0] * 8
    run_and_check(args, "sharp", weights=True)
    args[0] = args[0] * 0
    args[1] = args[1] * 0
    run_and_check(args, "flat", weights=True)


@pytest.mark.gpu
def test_nan_query_stays_in_its_row():
    from auto_gpu_kernel_b200 import paged_attention
    for n in (50, 30000):                                # one segment, and many that are joined
        args = list(make([n, 70], seed=11))
        args[0][0, 3] = float("nan")
        out, lse = paged_attention.run(*args, SCALE)
        assert torch.isnan(out[0, 3]).all() and torch.isnan(lse[0, 3])
        other = torch.ones(2, 16, dtype=torch.bool, device="cuda")
        other[0, 3] = False
        assert torch.isfinite(out[other]).all() and torch.isfinite(lse[other]).all()


@pytest.mark.gpu
def test_weights_in_place_from_nothing_and_repeatable():
    from auto_gpu_kernel_b200 import paged_attention
    args = make([5000, 64, 777], seed=12)
    width = args[5].shape[1] * PAGE
    fresh = torch.full((3, width), 9.0, device="cuda")
    out, lse = paged_attention.run(*args, SCALE, new_token_weights=fresh)
    for b, n in enumerate((5000, 64, 777)):
        total = fresh[b, :n].double().sum()
        assert abs(total - 16) <= 16 * 1e-4             # every row's weights add up to one
        assert (fresh[b, n:] == 9.0).all()
    twice = torch.where(fresh == 9.0, 0.0, fresh)
    again = twice.clone()
    o2, l2 = paged_attention.run(*args, SCALE, token_weights=again, new_token_weights=again)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    assert torch.equal(again, twice + twice)             # the same gain, and no other order of its sum


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes whose last pages are used (2^22 slots of 1024 bytes are 4 GiB)."""
    from auto_gpu_kernel_b200 import paged_attention, workspace
    pages = (1 << 16) + 40
    ckv = torch.zeros(pages, PAGE, 512, dtype=torch.bfloat16, device="cuda")
    kpe = torch.zeros(pages, PAGE, 64, dtype=torch.bfloat16, device="cuda")
    small = make([2000], seed=13)
    n = small[2].shape[0]
    ckv[-n:], kpe[-n:] = small[2], small[3]
    args = [small[0], small[1], ckv, kpe, small[4], small[5] + (pages - n)]
    out, lse = paged_attention.run(*args, SCALE)
    ref, rlse = paged_attention.run(*small, SCALE)
    assert workspace.check_status() == 0
    assert torch.equal(out, ref) and torch.equal(lse, rlse)


@pytest.mark.gpu
def test_other_stream_and_two_at_once():
    from auto_gpu_kernel_b200 import paged_attention
    a, b = make([3000, 10], seed=14), make([2500, 900], seed=15)
    ra, rb = paged_attention.run(*a, SCALE), paged_attention.run(*b, SCALE)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s):
            x = paged_attention.run(*a, SCALE)
        with torch.cuda.stream(t):
            y = paged_attention.run(*b, SCALE)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x[0], ra[0]) and torch.equal(x[1], ra[1])
        assert torch.equal(y[0], rb[0]) and torch.equal(y[1], rb[1])


@pytest.mark.gpu
def test_several_calls_in_a_row_on_changing_shapes():
    """Calls whose scratch buffers take one another's place, without a synchronisation in between."""
    from auto_gpu_kernel_b200 import paged_attention
    cases = [make([9000, 5], seed=30), make([700, 3, 0, 64], heads=64, seed=31), make([40], tokens=3, seed=32),
             make([20000], heads=20, seed=33), make([130] * 200, seed=34)]
    want = []
    for c in cases:
        want.append(paged_attention.run(*c, SCALE))
        torch.cuda.synchronize()
    got = [[paged_attention.run(*c, SCALE) for c in cases] for _ in range(8)]
    torch.cuda.synchronize()
    for round_ in got:
        for x, y in zip(round_, want):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.gpu
def test_on_a_device_that_is_not_current():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from auto_gpu_kernel_b200 import paged_attention
    args = make([900, 70], seed=35)
    want = paged_attention.run(*args, SCALE)
    there = paged_attention.run(*[t.to("cuda:1") for t in args], SCALE)
    assert torch.equal(want[0].cpu(), there[0].cpu()) and torch.equal(want[1].cpu(), there[1].cpu())


@pytest.mark.gpu
def test_captured_graphs_keep_their_own_workspaces():
    from auto_gpu_kernel_b200 import paged_attention
    cases = [make([3000, 10], seed=16), make([9000, 900, 64], seed=17)]
    want = [paged_attention.run(*c, SCALE) for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        width = c[5].shape[1] * PAGE
        grown = torch.zeros(len(c[4]), width, device="cuda")
        with torch.cuda.graph(g):
            res = paged_attention.run(*c, SCALE, token_weights=grown, new_token_weights=grown)
        graphs.append((g, res, grown))
    for _ in range(3):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (g, res, grown), w, c in zip(graphs, want, cases):
        assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])
        assert abs(float(grown.double().sum()) - 3 * 16 * len(c[4])) <= 1e-2
    # a graph follows new lengths and a longer cache than it was captured with
    g, res, _ = graphs[0]
    cases[0][4].copy_(torch.tensor([64, 1], dtype=torch.int32))
    g.replay()
    fresh = paged_attention.run(*cases[0], SCALE)
    torch.cuda.synchronize()
    assert torch.equal(res[0], fresh[0]) and torch.equal(res[1], fresh[1])


@pytest.mark.gpu
def test_refusals():
    from auto_gpu_kernel_b200 import paged_attention
    args = make([70, 5])

    def refuses(error, **at):
        a = list(args)
        kw = {}
        for k, v in at.items():
            if k in ("token_weights", "new_token_weights", "output", "lse"):
                kw[k] = v
            else:
                a[int(k[1:])] = v
        with pytest.raises(error):
            paged_attention.run(*a, SCALE, **kw)
    refuses(ValueError, a0=args[0].float())
    refuses(ValueError, a0=args[0][:, :, :500])
    refuses(ValueError, a1=args[1][:1])
    refuses(ValueError, a0=torch.cat([args[0], args[0][:1]]), a1=torch.cat([args[1], args[1][:1]]))
    refuses(ValueError, a0=args[0].transpose(0, 1).contiguous().transpose(0, 1), output=torch.empty_like(args[0]))
    refuses(ValueError, a2=args[2][:, :32])
    refuses(ValueError, a3=args[3][:-1])
    refuses(ValueError, a4=args[4].long())
    refuses(ValueError, a5=args[5].long())
    refuses(ValueError, a5=args[5].t().contiguous().t())
    refuses(RuntimeError, a4=args[4].cpu())
    refuses(RuntimeError, a2=args[2].cpu())
    refuses(ValueError, a0=args[0].repeat(1, 9, 1), a1=args[1].repeat(1, 9, 1))      # 144 heads
    w = torch.zeros(2, 128, device="cuda")
    refuses(ValueError, token_weights=w)
    refuses(ValueError, new_token_weights=w[:, :100])
    refuses(ValueError, new_token_weights=w.double())
    refuses(ValueError, new_token_weights=w[:1].expand(2, -1))
    big = torch.zeros(4, 128, device="cuda")
    refuses(ValueError, token_weights=big[:2], new_token_weights=big[1:3])
    refuses(RuntimeError, new_token_weights=w.cpu())
    refuses(ValueError, output=args[0])
    flat = torch.zeros(args[0].numel() + 512, dtype=torch.bfloat16, device="cuda")
    refuses(ValueError, a0=flat[:args[0].numel()].view(args[0].shape), output=flat[512:].view(args[0].shape))
    empty = paged_attention.run(args[0][:0], args[1][:0], *args[2:4], args[4][:0], args[5][:0], SCALE)
    assert empty[0].shape == (0, 16, 512)
    refuses(ValueError, a0=args[0][:0], a1=args[1][:0], new_token_weights=w)          # two requests, no query token
    none = paged_attention.run(*args[:5], args[5][:, :0], SCALE)
    assert (none[0] == 0).all() and torch.isinf(none[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,tokens", [(20, 1), (5, 4), (33, 2), (64, 1), (100, 1)])
def test_logits_of_padding_rows_are_not_stored(heads, tokens):
    """In blocks of 64 rows the scratch rows behind a request's last query row are not written; nobody reads them."""
    from auto_gpu_kernel_b200 import workspace
    lib = _lib.load()
    q_nope, q_pe, ckv, kpe, lens, table = make([300, 64, 0, 700], heads=heads, tokens=tokens, seed=70)
    table[3, 1] = -1                                     # a page that is left out
    batch, pages, rows = 4, table.shape[1], tokens * heads
    block = 64
    blocks = -(-rows // block)
    need = lib.dsa_paged_attn_workspace_bytes(batch, tokens, heads, pages, 1)
    scratch = torch.full((need,), 0xa5, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q_nope), torch.empty(q_nope.shape[:2], device="cuda")
    new = torch.zeros(batch, pages * PAGE, device="cuda")
    rc = workspace.call_on(0, lib.dsa_paged_attn, q_nope.data_ptr(), q_pe.data_ptr(), ckv.data_ptr(), kpe.data_ptr(), lens.data_ptr(),
                           table.data_ptr(), pages, SCALE, out.data_ptr(), lse.data_ptr(), None, 0, new.data_ptr(), pages * PAGE, batch,
                           tokens, heads, ckv.shape[0], pages, scratch.data_ptr(), need)
    assert rc == 0
    with pytest.raises(RuntimeError, match="block_table entry outside"):
        workspace.check_status()
    logits = scratch[need - 4 * batch * pages * blocks * block * PAGE:].view(torch.int32).view(batch, pages, blocks * block, PAGE)
    untouched = logits == -0x5a5a5a5b                    # bytes 0xa5
    assert untouched[:, :, rows:].all()
    for b, n in enumerate(lens.tolist()):
        held = -(-n // PAGE)
        assert not untouched[b, :held, :rows].any() and untouched[b, held:].all()
