"""Dense attention over long caches, by inputs whose result depends on every page: each page of a request has an output
column of its own (of 512, in turn) and logits that are whole numbers in base 2, so the expected values are sums of powers of two.
A page left out, counted twice or scaled by a wrong factor shows at any length.  Beside it a check of the rms error on
random inputs, which does not grow with the length as worst-case bounds do."""
import math

import pytest
import torch

import paged_oracle as po

PAGE = 64


def exponents(pages, kind, seed):
    """Base-2 logit of every page, whole numbers: `mixed` leaves a few heavy pages, `rising` refreshes the running maximum
    again and again (and falls for the rows of opposite sign)."""
    if kind == "mixed":
        gen = torch.Generator().manual_seed(seed)
        return torch.randint(-12, 13, (pages,), generator=gen).double()
    return torch.round(torch.arange(pages, dtype=torch.float64) * (100.0 / max(1, pages)))


def signs(heads):
    """What a head multiplies the exponents by: 0 (all tokens weigh the same), 1, -1, and so on."""
    return torch.tensor([(0.0, 1.0, -1.0)[h % 3] for h in range(heads)], dtype=torch.float64)


def expected(length, tokens, heads, e, times=None):
    """(out [tokens,heads,512], lse, gain [length]) of a request in 64 bits; `times` says how often each page counts."""
    pages = -(-length // PAGE)
    times = torch.ones(pages, dtype=torch.float64) if times is None else times
    out = torch.zeros(tokens, heads, 512, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    gain = torch.zeros(pages, PAGE, dtype=torch.float64)
    at = torch.arange(pages * PAGE).view(pages, PAGE)
    col = torch.arange(pages) % 512
    for i in range(tokens):
        seen = at < min(length, length - tokens + 1 + i)
        held = seen.sum(1).double() * times
        for h, s in enumerate(signs(heads).tolist()):
            w = torch.exp2(s * e[:pages])
            total = (held * w).sum()
            if total == 0:
                continue
            out[i, h] = torch.zeros(512, dtype=torch.float64).index_add_(0, col, held * w / total)
            lse[i, h] = torch.log2(total)
            gain += torch.where(seen, (w / total)[:, None], 0.0)
    return out, lse, gain.view(-1)[:length]


def check(out, lse, gain, want, length, rows, most, label=""):
    """Relative bounds, element by element (every term is positive).  A logit of E is off by 2^-22 E (its scale is a product
    of rounded numbers), a difference of two by as much again and a rounding; exp2 adds 2^-22: `eta`.  A weight within
    eta of a power of two rounds to that power.  Sums: at most length / 32 + 700 fp32 terms one after the other.  The
    output is rounded to bf16 (2^-8)."""
    w_out, w_lse, w_gain = want
    eta = (2.5 * most + 2) * 2.0 ** -22
    sums = (length / 32 + 700) * 2.0 ** -24
    tol = 2.0 ** -8 + 4 * eta + 2 * sums
    err = (out.double().cpu() - w_out).abs()
    assert (err <= tol * w_out).all(), f"{label}: output off by {(err / (tol * w_out).clamp_min(1e-300)).max():.2f} of its bound"
    lse = lse.double().cpu()
    none = torch.isinf(w_lse)
    assert torch.equal(torch.isinf(lse), none), label
    bound = (2 * eta + sums) / math.log(2.0) + 2.0 ** -22 * w_lse[~none].abs()
    err = (lse - w_lse)[~none].abs()
    assert (err <= bound).all(), f"{label}: lse off by {(err / bound).max():.2f} of its bound"
    if gain is not None:
        tol = 4 * eta + 2 * sums + (rows + 40) * 2.0 ** -23
        err = (gain.double().cpu() - w_gain).abs()
        assert (err <= tol * w_gain).all(), f"{label}: weights off by {(err / (tol * w_gain).clamp_min(1e-300)).max():.2f} of their bound"


def make(lens, heads, tokens, kind, seed, device="cuda"):
    need = [-(-n // PAGE) for n in lens]
    pages = sum(need) + 1
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    ckv = torch.full((pages, PAGE, 512), float("nan"), dtype=torch.bfloat16)
    kpe = torch.full((pages, PAGE, 64), float("nan"), dtype=torch.bfloat16)
    e = [exponents(k, kind, seed + b) for b, k in enumerate(need)]
    at = 0
    for b, (n, k) in enumerate(zip(lens, need)):
        mine = perm[at:at + k]
        at += k
        table[b, :k] = mine
        ckv[mine], kpe[mine] = 0.0, 0.0
        ckv[mine, :, torch.arange(k) % 512] = 1.0
        kpe[mine, :, 0] = e[b].to(torch.bfloat16)[:, None]
        if n % PAGE:
            ckv[mine[-1], n % PAGE:] = float("nan")
            kpe[mine[-1], n % PAGE:] = float("inf")
    rows = len(lens) * tokens
    q_nope = torch.zeros(rows, heads, 512, dtype=torch.bfloat16)
    q_pe = torch.zeros(rows, heads, 64, dtype=torch.bfloat16)
    q_pe[:, :, 0] = signs(heads).to(torch.bfloat16)
    args = (q_nope, q_pe, ckv, kpe, torch.tensor(lens, dtype=torch.int32), table)
    return [t.to(device) for t in args], e


def random_error(out, want):
    """Rms error of an output of random inputs over its rms.  A bf16 rounding is uniform over a step of at most 2^-7 of the
    value: at most 2^-7 / sqrt(12) of the output's rms; the softmax weights are rounded alike, independently of one
    another, and rows of zero mean add up as they do in the output.  Both: 0.0032; the fp32 parts are far below 0.0003."""
    return float((out.double().cpu() - want.cpu()).square().mean().sqrt() / want.square().mean().sqrt().cpu())


RANDOM_BOUND = 0.0035


# ------------------------------------------------------------------------------------------ CPU
def rounded(want):
    return want[0].to(torch.bfloat16), want[1].float(), want[2].float()


@pytest.mark.parametrize("length,kind", [(70001, "mixed"), (70001, "rising"), (20000, "mixed"), (700, "rising")])
def test_the_check_sees_every_page(length, kind):
    pages = -(-length // PAGE)
    e = exponents(pages, kind, 1)
    want = expected(length, 1, 6, e)
    check(*rounded(want), want, length, 6, 100)

    def caught(times, gains=True):
        wrong = rounded(expected(length, 1, 6, e, times))
        with pytest.raises(AssertionError):
            check(*wrong[:2], wrong[2] if gains else None, want, length, 6, 100)
        with pytest.raises(AssertionError):              # the output alone shows it, too
            check(wrong[0], want[1], None, want, length, 6, 100)
    for j in sorted({0, 1, pages // 2, pages - 2}):
        for factor in (0.0, 2.0, 0.5):
            times = torch.ones(pages, dtype=torch.float64)
            times[j] = factor
            caught(times)
            caught(times, gains=False)
    if pages > 100:
        for factor in (0.0, 0.97):                       # a partial result lost, or joined with a wrong factor
            times = torch.ones(pages, dtype=torch.float64)
            times[50:58] = factor
            caught(times)


def test_the_plain_form_gives_the_expected_values():
    """The closed form against the 64-bit attention on the same inputs, drafted tokens and an empty request among them."""
    lens, heads, tokens = [700, 2, 0, 129], 4, 3
    args, e = make(lens, heads, tokens, "mixed", 3, device="cpu")
    args[2] = torch.nan_to_num(args[2])
    args[3] = torch.nan_to_num(args[3], posinf=0.0)
    out, lse, grown, _, _ = po.attend(*args, math.log(2.0), torch.zeros(4, args[5].shape[1] * PAGE))
    for b, n in enumerate(lens):
        want = expected(n, tokens, heads, e[b])
        mine = slice(b * tokens, (b + 1) * tokens)
        assert torch.allclose(out[mine], want[0], rtol=1e-12) and torch.allclose(lse[mine], want[1], rtol=1e-12)
        assert torch.allclose(grown[b, :n], want[2], rtol=1e-12)


def test_the_rms_check_sees_a_page():
    gen = torch.Generator().manual_seed(4)
    n = 30000
    q, k = torch.randn(4, 576, generator=gen, dtype=torch.float64), torch.randn(n, 576, generator=gen, dtype=torch.float64)
    p = torch.softmax(q @ k.t() / math.sqrt(192.0), 1)
    want = p @ k[:, :512]
    kernel = (p.to(torch.bfloat16).double() @ k[:, :512]).to(torch.bfloat16)
    assert random_error(kernel, want) <= RANDOM_BOUND
    p[:, 6400:6464] = 0
    assert random_error((p @ k[:, :512]).to(torch.bfloat16), want) > RANDOM_BOUND


# ------------------------------------------------------------------------------------------ GPU
LONG = [[70001], [40000, 1, 25000, 64], [30000, 29999, 30001], [9000, 7, 130, 64, 0, 12345, 8000, 3],
        [2000 + 37 * b for b in range(100)], [33000]]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mixed", "rising"])
@pytest.mark.parametrize("heads,tokens", [(16, 1), (5, 3), (16, 4), (33, 1), (128, 1)])
@pytest.mark.parametrize("lens", LONG, ids=lambda v: f"{len(v)}x{max(v)}")
def test_every_page_counts_once(lens, heads, tokens, kind):
    """Up to 148 partial results per request, joined by every number of groups, in blocks of 16 and of 64 rows."""
    from auto_gpu_kernel_b200 import paged_attention, workspace
    args, e = make(lens, heads, tokens, kind, seed=len(lens) + heads)
    grown = torch.zeros(len(lens), args[5].shape[1] * PAGE, device="cuda")
    out, lse = paged_attention.run(*args, math.log(2.0), new_token_weights=grown)
    plain = paged_attention.run(*args, math.log(2.0))
    assert workspace.check_status() == 0
    assert torch.equal(plain[0], out) and torch.equal(plain[1], lse)      # with and without weights
    out, lse, grown = out.cpu(), lse.cpu(), grown.cpu()
    for b, n in enumerate(lens):
        mine = slice(b * tokens, (b + 1) * tokens)
        want = expected(n, tokens, heads, e[b])
        check(out[mine], lse[mine], grown[b, :n], want, n, tokens * heads, 100, f"request {b} of {n} tokens")
        assert (grown[b, n:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,most", [(100, 500), (148, 512), (300, 250), (700, 512)])
@pytest.mark.parametrize("heads", [16, 48])
def test_every_page_counts_once_in_short_requests(batch, most, heads):
    """Requests that stay whole, one or several to a CTA."""
    test_every_page_counts_once([1 + (37 * b) % most for b in range(batch)], heads, 1, "mixed")


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [16, 64])
@pytest.mark.parametrize("length", [30000, 70001])
def test_rms_error_of_a_long_request(length, heads):
    from test_paged_attention import SCALE
    from test_paged_attention import make as random_case
    from auto_gpu_kernel_b200 import paged_attention
    args = random_case([length], heads=heads, seed=50)
    fresh = torch.zeros(1, args[5].shape[1] * PAGE, device="cuda")
    out, lse = paged_attention.run(*args, SCALE, new_token_weights=fresh)
    want = po.attend(*args, SCALE)
    error = random_error(out, want[0])
    assert error <= RANDOM_BOUND, f"rms error {error:.5f}"
    # a logit is added up in 36 steps of 16 products from partial sums below 12 (in base 2): 36 * 12 * 2^-23 = 5e-5 at most; the
    # sums of the weights and the rounding of an lse below 32 add less than 1e-5.  Every row's weights add up to one
    assert (lse.double() - want[1]).abs().max() <= 1e-4
    assert abs(float(fresh.double().sum()) - heads) <= 1e-4 * heads
