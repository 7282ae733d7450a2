"""The operators as a serving loop runs them together: rotary append -> dense attention with accumulated weights ->
eviction to new pages -> the indexer and the sparse attention on what was kept -> another dense step."""
import math

import pytest
import torch

import paged_oracle as po

SCALE = 1.0 / math.sqrt(192.0)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_append_attend_evict_and_go_on(graph):
    from auto_gpu_kernel_b200 import cache_evict, indexer, inputs, paged_attention, rotary, sparse_attention, workspace
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(0)
    lens, budget, steps = [700, 130, 2999], 256, 3
    batch = len(lens)
    per, fresh = 3100 // 64 + 1, budget // 64 + 1
    pages = batch * (per + fresh)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(dev)
    table, new_table = perm[:batch * per].view(batch, per), perm[batch * per:].view(batch, fresh)
    half = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=torch.bfloat16)
    ckv, kpe = half(pages, 64, 512), half(pages, 64, 64)
    keys = inputs.pack_index_pages(torch.randn(pages, 64, 128, generator=gen, device=dev))
    inv_freq = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(dev)
    axes = rotary.sections(16, 8, 8)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    weights = torch.zeros(batch, per * 64, device=dev)

    feed = dict(q_nope=half(batch, 16, 512), q_pe=half(batch, 16, 64), ckv=half(batch, 512), kpe=half(batch, 64),
                positions=torch.zeros(3, batch, dtype=torch.int32, device=dev),
                slots=torch.zeros(batch, dtype=torch.int32, device=dev))

    def step():
        q = rotary.append(feed["q_pe"], feed["ckv"], feed["kpe"], feed["positions"], inv_freq, axes, feed["slots"], ckv, kpe)
        out, lse = paged_attention.run(feed["q_nope"], q, ckv, kpe, seq_lens, table, SCALE, token_weights=weights,
                                       new_token_weights=weights)
        return q, out, lse

    if graph:
        feed["slots"].fill_(-1)            # the warm-up changes no cache row
        step()
        weights.zero_()
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            result = step()
        weights.zero_()
    for i in range(steps):
        seq_lens += 1
        for name in ("q_nope", "q_pe", "ckv", "kpe"):
            feed[name].copy_(half(*feed[name].shape))
        feed["positions"].copy_(seq_lens[None].expand(3, -1) + torch.tensor([[0], [3], [5]], device=dev))
        feed["slots"].copy_(torch.stack([table[b, (n + i) // 64] * 64 + (n + i) % 64 for b, n in enumerate(lens)]))
        before = weights.clone()
        if graph:
            captured.replay()
            q, out, lse = result
        else:
            q, out, lse = step()
        want = po.attend(feed["q_nope"], q, ckv, kpe, seq_lens, table, SCALE, before)
        po.check_attend(out, lse, want, max(lens) + i + 1, weights, before, 16, f"step {i}")
    held = torch.arange(weights.shape[1], device=dev)[None] < seq_lens[:, None]
    assert (weights[~held] == 0).all()

    short, kept_weights, kept = cache_evict.run(weights, seq_lens, table, new_table, budget, ckv, kpe, keys, keep_first=4,
                                                keep_last=32)
    assert short.tolist() == [256, 133, 256]
    for b, n in enumerate(seq_lens.tolist()):
        mine = po.evict_choice(weights[b], n, budget, 4, 32)
        assert kept[b, :len(mine)].tolist() == mine

    # what was kept reads back through both attentions: the sparse one sees all of it, being within its 2048 slots
    dense, dense_lse = paged_attention.run(feed["q_nope"], q, ckv, kpe, short, new_table, SCALE)
    topk = indexer.run(torch.randn(batch, 64, 128, generator=gen, device=dev).to(torch.float8_e4m3fn), keys,
                       torch.randn(batch, 64, generator=gen, device=dev), short, new_table)
    sparse, sparse_lse = sparse_attention.run(feed["q_nope"], q, ckv, kpe, topk, SCALE)
    want = po.attend(feed["q_nope"], q, ckv, kpe, short, new_table, SCALE)
    po.check_attend(dense, dense_lse, want, 256, label="after eviction, dense")
    po.check_attend(sparse, sparse_lse, want, 256, label="after eviction, sparse")

    # and the loop goes on from the short caches: the weights that were kept go on growing
    grown = torch.zeros(batch, fresh * 64, device=dev)
    grown[:, :budget] = kept_weights
    feed["slots"].copy_(torch.stack([new_table[b, n // 64] * 64 + n % 64 for b, n in enumerate(short.tolist())]))
    short += 1
    before = grown.clone()
    q = rotary.append(feed["q_pe"], feed["ckv"], feed["kpe"], feed["positions"], inv_freq, axes, feed["slots"], ckv, kpe)
    out, lse = paged_attention.run(feed["q_nope"], q, ckv, kpe, short, new_table, SCALE, token_weights=grown, new_token_weights=grown)
    want = po.attend(feed["q_nope"], q, ckv, kpe, short, new_table, SCALE, before)
    po.check_attend(out, lse, want, 257, grown, before, 16, "after eviction, next step")
    assert workspace.check_status() == 0
