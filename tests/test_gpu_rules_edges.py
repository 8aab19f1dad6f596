"""The rules between logits and token where their ordinary tests do not go: lists of biases with repeated ids."""
import numpy as np
import pytest

from test_gpu_rules import F, check, make

pytestmark = pytest.mark.gpu


def repeated_ids(g, rows, vocab, entries, pattern):
    """Bias ids [rows, entries], of which each stands there once, twice, or many times."""
    ids = np.empty((rows, entries), np.int64)
    for r in range(rows):
        if pattern == "twice":
            some = g.permutation(max(vocab, entries))[:(entries + 1) // 2] % vocab
            ids[r] = g.permutation(np.concatenate([some, some])[:entries])
        elif pattern == "one often":
            ids[r] = np.where(g.random(entries) < 0.6, g.integers(0, vocab), g.integers(0, vocab, entries))
        elif pattern == "runs":
            ids[r] = np.sort(g.integers(0, max(1, vocab // 3), entries))
        else:  # one id twice, at the ends of the list
            ids[r] = g.permutation(max(vocab, entries))[:entries] % vocab
            ids[r, -1] = ids[r, 0]
    return ids.astype(np.int32)


@pytest.mark.parametrize("pattern", ["twice", "one often", "runs", "ends"])
@pytest.mark.parametrize("rows,vocab,entries,history", [
    (3, 5000, 2000, 300),       # a count for every token of the chunk
    (2, 131072, 9000, 0),       # a cluster per row, slots
    (1, 140000, 30000, 700),    # several chunks per CTA
    (300, 1000, 256, 40),       # many rows
    (1, 33, 65535, 5)])
def test_repeated_biases(svl_lib, rows, vocab, entries, history, pattern):
    """Each token's biases are added in the list's order, whichever repeat."""
    g, r = make(rows, vocab, rows + entries, history=history, dense=True, masks=2)
    r["bias_ids"] = repeated_ids(g, rows, vocab, entries, pattern)
    if entries <= vocab:
        r["bias_ids"][g.random((rows, entries)) < 0.05] = -1  # pads in between
    r["bias_values"] = (g.standard_normal((rows, entries)) * (3 if entries < 10000 else 0.01)).astype(F)
    logits = (4 * g.standard_normal((rows, vocab))).astype(F)
    check(logits, r, "f32", offset=rows % 4)
    check(logits, r, "bf16", offset=3, in_place=True)


def shortest(call):
    """Device time of a call, ms: the shortest of some runs of ten."""
    import torch
    best = 1e9
    for _ in range(6):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(10):
            call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / 10)
    return best


@pytest.mark.parametrize("rows,vocab,entries", [(1, 131072, 16384), (64, 32000, 4096)])
def test_a_repeated_id_costs_no_more_than_the_list(svl_lib, rows, vocab, entries):
    """The time grows with the list, not with its square, when an id stands there twice: one more pass over the
    list. (It was 60 times as long where every biased token then walked the list.)"""
    import torch

    import svl
    g = np.random.default_rng(1)
    logits = torch.randn(rows, vocab, device="cuda")
    once = np.stack([g.permutation(vocab)[:entries] for _ in range(rows)]).astype(np.int32)
    twice = once.copy()
    twice[:, -1] = twice[:, 0]
    values = torch.randn(rows, entries, device="cuda")

    def time(ids):
        ids = torch.from_numpy(ids).cuda()
        return shortest(lambda: svl.logits_rules(logits, bias_ids=ids, bias_values=values))

    plain, repeated = time(once), time(twice)
    print(f"{rows} x {vocab}, {entries} biases: {plain * 1e3:.1f} us, {repeated * 1e3:.1f} with an id twice")
    assert repeated < 8 * plain


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_lists_leave_room_for_fewer_rows_at_once(svl_lib, dtype):
    """Rows are shared among CTAs by how many run at once with the shared memory that their lists take: twice the
    rows take no more than about twice the time. (2.9 times f32, 2.5 bf16, where the plan left the lists out.)"""
    import torch

    import svl
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    vocab, said = 50257, 6000
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(256, vocab, device="cuda", generator=g).to(t)
    history = torch.randint(0, vocab, (256, said), device="cuda", dtype=torch.int32, generator=g)
    lengths, penalty = torch.full((256,), said, dtype=torch.int32, device="cuda"), torch.full((256,), 1.5, device="cuda")
    rules = lambda n: svl.logits_rules(logits[:n], history=history[:n], lengths=lengths[:n], repetition=penalty[:n])  # noqa: E731
    half, all_ = shortest(lambda: rules(128)), shortest(lambda: rules(256))
    print(f"{dtype}: 128 rows {half * 1e3:.1f} us, 256 rows {all_ * 1e3:.1f}")
    assert all_ < 2.1 * half
    want, token = rules(128)
    got, tokens = rules(256)
    assert torch.equal(got[:128], want) and torch.equal(tokens[:128], token)
