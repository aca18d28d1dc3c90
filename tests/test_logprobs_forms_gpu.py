"""Log probabilities read inside the head's product (csrc/head_logprobs.cu): rows whose list cannot hold what is due, rows in several pieces, captured calls."""

import pytest
import torch

from plain_packed import logprobs
from test_logprobs_gpu import DEV, check, ops_for

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def on_a_grid(rows, width, V, seed):
    """Numbers whose sums are exact in float32 in any order: the alternatives are a fact."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = ((torch.randn(rows, width, generator=g, device=DEV) * 8).round() / 8).clamp(-6, 6)
    table = ((torch.randn(V, width, generator=g, device=DEV) * 20).round() / 512).clamp(-0.49, 0.49)
    return x, table, torch.randint(V, (rows,), generator=g, device=DEV).int()


def counts_of_lists(ops):
    """Notes the row counts of the lists that a call fills; entries beyond 2,048 did not fit."""
    noted, plain = [], ops.empty

    def empty(shape, dtype, device):
        tensor = plain(shape, dtype, device)
        if dtype is torch.int64:
            noted.append(len(shape))
        elif dtype is torch.int32 and noted and len(noted) == 1:
            noted.append(tensor)                                           # (the first int32 tensor behind the lists)
        return tensor

    ops.empty = empty
    return noted


@pytest.mark.parametrize("kind", ["sampled tokens least", "sampled tokens no numbers", "few sampled numbers", "rows of minus infinity"])
@pytest.mark.parametrize("rows,V", [(128, 20000), (300, 20000), (64, 50257)])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_rows_that_are_formed_again(kind, rows, V, top):
    """A sample that says nothing, or that bounds nothing: the list overflows, or holds fewer than are due, and the row is formed once more, token by token."""
    ops, width = ops_for(BF16), 64
    x, table, targets = on_a_grid(rows, width, V, rows)
    sampled = torch.arange(V, device=DEV) % ops.sample_every(V, top) == 0
    x[:, 0] = 4.0
    table[:, 0] = 0.0
    if kind == "sampled tokens least":
        table[:, 0] = torch.where(sampled, -8.0, 8.0)
    x, table = x.to(BF16), table.to(BF16)
    if kind == "sampled tokens no numbers":
        table[sampled, 3] = float("nan")
    elif kind == "few sampled numbers":
        some = sampled.nonzero()[top // 2:, 0]
        table[some, 3] = float("nan")
    elif kind == "rows of minus infinity":
        # all but a few tokens have probability 0: the bound is minus infinity
        x[:, 1] = 1.0
        table[17:, 1] = float("-inf")
        table[sampled, 1] = float("-inf")
    assert ops.fused_head_ok(x, table, top)
    noted = counts_of_lists(ops)
    found = ops.head_logprobs(x, table, targets, top)
    del ops.empty
    count = noted[1]
    assert ((count > 2048) | (count < top)).any() or kind == "rows of minus infinity"      # (that is, the branch is reached)
    logits = x.double() @ table.double().t()
    if kind in ("sampled tokens no numbers", "few sampled numbers"):
        assert found.logprob.isnan().all() and found.entropy.isnan().all() and found.top_logprobs.isnan().all()
        order = torch.sort(logits.nan_to_num(nan=float("-inf")), dim=1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(found.top_ids.long(), order)
    elif kind == "rows of minus infinity":
        given, entropy, best, ids = logprobs(logits.cpu(), targets.cpu(), top)
        assert torch.equal(found.top_ids.cpu(), ids) and (found.logprob.cpu()[given == float("-inf")] == float("-inf")).all()
        assert (found.entropy.cpu() - entropy.float()).abs().max() < 1e-4 if not entropy.isnan().any() else True
        assert ((found.top_logprobs.cpu() - best.float()).abs() < 1e-4)[best > float("-inf")].all()
        assert torch.equal(found.top_logprobs.cpu() == float("-inf"), best == float("-inf"))
    else:
        check(found, logits, targets, top)


@pytest.mark.parametrize("rows,V,top", [(128, 131072, 32), (64, 262144, 20), (64, 400001, 1), (64, 100003, 7)])
def test_large_vocabularies(rows, V, top):
    """The sample grows with the vocabulary and the alternatives: what lies beyond its bound fits the lists."""
    ops = ops_for(BF16)
    x, table, targets = on_a_grid(rows, 64, V, V)
    x, table = x.to(BF16), table.to(BF16)
    assert ops.fused_head_ok(x, table, top)
    noted = counts_of_lists(ops)
    found = ops.head_logprobs(x, table, targets, top)
    del ops.empty
    assert int(noted[1].max()) <= 2048 and int(noted[1].min()) >= top
    check(found, x.double() @ table.double().t(), targets, top)


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("most", [128, 200])
def test_pieces_of_many_rows(top, most):
    """Rows in pieces of FUSED_HEAD_MOST, the last one short, from a step's arena and without one."""
    from pagedserve_b200.kernels.ops import StepArena

    ops = ops_for(BF16)
    x, table, targets = on_a_grid(517, 96, 9000, 3)
    x, table = x.to(BF16), table.to(BF16)
    whole = ops.head_logprobs(x, table, targets, top)
    logits = x.double() @ table.double().t()
    check(whole, logits, targets, top)
    ops.FUSED_HEAD_MOST = most
    check(ops.head_logprobs(x, table, targets, top), logits, targets, top)
    ops.arena = StepArena()
    ops.empty((1000,), torch.float32, x.device)
    before = ops.arena.mark()
    check(ops.head_logprobs(x, table, targets, top), logits, targets, top)
    assert ops.arena.mark() == before                                      # (a piece's scratch is the next one's)


@pytest.mark.parametrize("top", [0, 4])
def test_a_captured_fused_head(top):
    """Captured on a side stream and replayed with other rows."""
    ops, rows, V = ops_for(BF16), 150, 9001
    x, table, targets = on_a_grid(rows, 128, V, 7)
    x, table = x.to(BF16), table.to(BF16)
    assert ops.fused_head_ok(x, table, top)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.head_logprobs(x, table, targets, top)
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        found = ops.head_logprobs(x, table, targets, top)
        graph.capture_end()
    side.synchronize()
    x.copy_(x.flip(0))
    targets.copy_(targets.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    check(found, x.double() @ table.double().t(), targets, top)
    del graph


@pytest.mark.parametrize("rows,width,V", [(130, 768, 20000), (128, 200, 9000)])
def test_tokens_with_the_same_row_of_the_table(rows, width, V):
    """Equal logits whose sums are rounded: the lower tokens, in order, whichever of them the sample holds."""
    ops, kinds, top = ops_for(BF16), 97, 32
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(rows, width, generator=g, device=DEV).to(BF16)
    base = (torch.randn(kinds, width, generator=g, device=DEV) / 4).to(BF16)
    table = base[torch.arange(V, device=DEV) % kinds].contiguous()
    assert ops.fused_head_ok(x, table, top)
    found = ops.head_logprobs(x, table, torch.zeros(rows, dtype=torch.int32, device=DEV), top)
    two, order = (x.double() @ base.double().t()).topk(2, dim=1)
    # float32 sums of `width` products are off by at most width * 2^-24 of the products' sizes: beyond that the best kind is a fact
    clear = two[:, 0] - two[:, 1] > 2 * width * 2.0 ** -24 * (x.double().abs() @ base.double().abs().t()).amax(1)
    assert clear.sum() > rows * 0.9
    assert torch.equal(found.top_ids[clear].long(), (order[:, :1] + kinds * torch.arange(top, device=DEV))[clear])
