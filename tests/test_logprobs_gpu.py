"""Log probabilities of given tokens, entropies and alternatives (csrc/logprobs.cu) against 64 bits, from logits and from the head's rows."""

import math

import pytest
import torch

from plain_packed import logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops_for(dtype=torch.float32):
    from test_kernels_gpu import ops_for as make

    return make(dtype)


def check(found, logits, targets, top, slack=0.0):
    """``slack``: how far the logits themselves may be off."""
    given, entropy, best, ids = logprobs(logits.double().cpu(), targets.cpu(), top)
    V = logits.shape[1]
    # sums of V weights in parts of at most 256 and 8 levels above them, exponentials good to 2^-20 each, in float32; the difference x - m is rounded
    # to 2^-24 of itself
    span = (logits.double().amax(1) - torch.where(logits.isinf(), logits.amax(1, keepdim=True), logits).double().amin(1)).cpu()
    step = 2.0 ** -19 + 2.0 ** -24 * (min(V, 264) + span) + 4 * slack
    assert (((found.logprob.cpu().double() - given).abs() <= step * (1 + given.abs())) | (found.logprob.cpu() == given)).all()       # (-infinity)
    assert ((found.entropy.cpu().double() - entropy).abs() <= step * (4 + 2 * math.log(V) + entropy)).all()
    assert torch.equal(found.top_ids.cpu(), ids)
    assert (((found.top_logprobs.cpu().double() - best).abs() <= step[:, None] * (1 + best.abs())) | (found.top_logprobs.cpu() == best)).all()


@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (2, 33), (5, 255), (4, 2048), (7, 2049), (3, 4097), (9, 50257), (200, 8200), (500, 5000), (1000, 4100)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_sizes(rows, V, top):
    ops, top = ops_for(), min(top, V)
    g = torch.Generator(device=DEV).manual_seed(rows + V)
    wide = torch.randn(rows, V + 3, generator=g, device=DEV) * 4
    logits = wide[:, 1:1 + V]                                           # rows that start anywhere
    targets = torch.randint(V, (rows,), generator=g, device=DEV).int()
    check(ops.token_logprobs(logits, targets, top), logits, targets, top)


@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "blocks", "one large", "tiny and huge", "half gone"])
@pytest.mark.parametrize("V", [600, 12345])
def test_orders_and_ties(kind, V):
    """Equal logits (the lower index first), rows in which every number beats those in front, groups that hold all the largest."""
    ops = ops_for()
    g = torch.Generator(device=DEV).manual_seed(1)
    i = torch.arange(V, device=DEV).float()
    row = {"equal": torch.full((V,), 1.5, device=DEV), "few values": torch.randint(3, (V,), generator=g, device=DEV).float(), "rising": i / 100,
           "falling": -i / 100, "blocks": ((i % 2048) < 40) * 5.0 + torch.rand(V, generator=g, device=DEV), "one large": (i == V - 1) * 80.0,
           "tiny and huge": torch.where(i % 2 == 0, 3e38, -3e38), "half gone": torch.where(i % 2 == 0, float("-inf"), i / V)}[kind]
    logits = torch.stack([row, row.flip(0), row * 0 - 0.0 if kind == "equal" else row])
    targets = torch.tensor([0, V - 1, V // 2], dtype=torch.int32, device=DEV)
    check(ops.token_logprobs(logits, targets, 32), logits, targets, 32)


def test_rows_that_say_nothing():
    """A NaN or +infinity makes a row's numbers NaN and no other's; minus infinity is probability 0; NaN comes last in the order."""
    ops, V = ops_for(), 5000
    logits = torch.randn(6, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    logits[1, 4000] = float("nan")
    logits[2, 100] = float("inf")
    logits[3] = float("-inf")
    logits[4] = float("nan")
    logits[4, 4321] = 1.0
    found = ops.token_logprobs(logits, torch.zeros(6, dtype=torch.int32, device=DEV), 4)
    for name in ("logprob", "entropy"):
        assert getattr(found, name).isnan().tolist() == [False, True, True, True, True, False]
    assert found.top_ids[2, 0] == 100 and found.top_ids[3].tolist() == [0, 1, 2, 3] and found.top_ids[4].tolist() == [4321, 0, 1, 2]
    assert 4000 not in found.top_ids[1].tolist()
    check(type(found)(*(t[[0, 5]] for t in found)), logits[[0, 5]], torch.zeros(2, dtype=torch.int32), 4)
    ops.status_flag(logits.device)
    assert int(ops.status.item()) == 0


def test_tokens_outside_and_none():
    ops, V = ops_for(), 3000
    logits = torch.randn(4, V, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    found = ops.token_logprobs(logits, torch.tensor([-1, 5, -1, 2999], dtype=torch.int32, device=DEV), 1, status)
    assert found.logprob[[0, 2]].tolist() == [0.0, 0.0] and int(status.item()) == 0 and (found.logprob[[1, 3]] < 0).all()
    found = ops.token_logprobs(logits, torch.tensor([-2, 3000, 2 ** 31 - 1, 0], dtype=torch.int32, device=DEV), 1, status)
    assert found.logprob.isnan().tolist() == [True, True, True, False] and int(status.item()) != 0 and found.entropy.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width,V", [(1, 64, 700), (5, 768, 50257), (33, 96, 5000), (129, 64, 1031), (300, 200, 32000), (400, 768, 50257), (130, 1600, 2000)])
@pytest.mark.parametrize("top", [0, 3, 32])
def test_from_the_heads_rows(dtype, rows, width, V, top):
    """Numbers on a grid whose sums are exact in float32 in any order: the alternatives are a fact."""
    ops = ops_for(dtype)
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = ((torch.randn(rows, width + 8, generator=g, device=DEV) * 8).round() / 8).clamp(-6, 6).to(dtype)[:, :width]
    table = ((torch.randn(V, width, generator=g, device=DEV) * 20).round() / 512).clamp(-0.49, 0.49).to(dtype)
    targets = torch.randint(V, (rows,), generator=g, device=DEV).int()
    logits = x.double() @ table.double().t()
    check(ops.head_logprobs(x, table, targets, top), logits, targets, top)


@pytest.mark.parametrize("kind", ["zero rows", "rising", "every other sampled", "one token", "infinite"])
@pytest.mark.parametrize("rows", [96, 300])
def test_heads_that_fool_a_sample(kind, rows):
    """Rows whose logits are all equal, rise with the token, or are least at every token that a regular sample meets; a table with a row that is not finite."""
    ops, width, V, top = ops_for(torch.bfloat16), 64, 20000, 20
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = ((torch.randn(rows, width, generator=g, device=DEV) * 8).round() / 8).clamp(-6, 6)
    table = ((torch.randn(V, width, generator=g, device=DEV) * 20).round() / 512).clamp(-0.49, 0.49)
    i = torch.arange(V, device=DEV)
    if kind == "zero rows":
        x[::3] = 0
    elif kind == "rising":
        table[:, 0], x[:, 0] = (i // 100 * 0.25), 1.0                   # (multiples of 1/4 up to 50: exact in bfloat16)
    elif kind == "every other sampled":
        table[:, 0], x[:, 0] = torch.where(i % (V // 2048) == 0, -8.0, 8.0), 4.0
    elif kind == "one token":
        table[V - 1, 0], x[:, 0] = 16.0, 4.0
    x, table = x.bfloat16(), table.bfloat16()
    if kind == "infinite":
        table[777, 5] = float("inf")
        x[:, 5] = torch.where(torch.arange(rows, device=DEV) % 2 == 0, -1.0, 1.0).bfloat16()       # minus infinity in even rows, infinity in odd ones
    targets = torch.randint(V, (rows,), generator=g, device=DEV).int()
    found = ops.head_logprobs(x, table, targets, top)
    logits = x.double() @ table.double().t()
    if kind == "infinite":
        assert found.logprob[1::2].isnan().all() and found.entropy[1::2].isnan().all() and (found.top_ids[1::2, 0] == 777).all()
        found, logits, targets = type(found)(*(t[::2] for t in found)), logits[::2], targets[::2]
    check(found, logits, targets, top)


@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("rows,width,V", [(15, 64, 8192), (16, 64, 8192), (17, 200, 41000), (47, 96, 40001), (48, 96, 40001), (127, 64, 9001), (128, 72, 9001)])
def test_rows_around_the_choice_of_a_form(rows, width, V, top):
    """Read inside the product or from logits: numbers on a grid whose sums are exact, as above."""
    ops = ops_for(torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(rows + width)
    x = ((torch.randn(rows, width, generator=g, device=DEV) * 8).round() / 8).clamp(-6, 6).bfloat16()
    table = ((torch.randn(V, width, generator=g, device=DEV) * 20).round() / 512).clamp(-0.49, 0.49).bfloat16()
    targets = torch.randint(-1, V, (rows,), generator=g, device=DEV).int()
    assert ops.fused_head_ok(x, table, top) == (rows >= (16 if not top else 48 if V > 40000 else 128))
    check(ops.head_logprobs(x, table, targets, top), x.double() @ table.double().t(), targets, top)


@pytest.mark.parametrize("rows,width,V", [(96, 768, 20000), (300, 200, 9000), (1500, 1600, 8500)])
def test_tokens_with_the_same_row_of_the_table(rows, width, V):
    """Equal logits whose sums are rounded: the lower tokens, in order, whichever of them a sample of the vocabulary holds."""
    ops, kinds, top = ops_for(torch.bfloat16), 97, 32
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(rows, width, generator=g, device=DEV).bfloat16()
    base = (torch.randn(kinds, width, generator=g, device=DEV) / 4).bfloat16()
    table = base[torch.arange(V, device=DEV) % kinds].contiguous()
    found = ops.head_logprobs(x, table, torch.zeros(rows, dtype=torch.int32, device=DEV), top)
    logits = x.double() @ base.double().t()
    two, order = logits.topk(2, dim=1)
    # float32 sums of `width` products are off by at most width * 2^-24 of the products' sizes: beyond that the best kind is a fact
    clear = two[:, 0] - two[:, 1] > 2 * width * 2.0 ** -24 * (x.double().abs() @ base.double().abs().t()).amax(1)
    assert clear.sum() > rows * 0.9
    want = order[:, :1] + kinds * torch.arange(top, device=DEV)
    assert torch.equal(found.top_ids[clear].long(), want[clear])
    assert (found.top_logprobs == found.top_logprobs[:, :1])[clear].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_captured_head(dtype):
    """Captured on a side stream and replayed with other rows."""
    ops, rows, width, V = ops_for(dtype), 150, 128, 3001
    g = torch.Generator(device=DEV).manual_seed(7)
    x = ((torch.randn(rows, width, generator=g, device=DEV) * 8).round() / 8).to(dtype)
    table = ((torch.randn(V, width, generator=g, device=DEV) * 20).round() / 512).to(dtype)
    targets = torch.randint(V, (rows,), generator=g, device=DEV).int()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.head_logprobs(x, table, targets, 4)
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        found = ops.head_logprobs(x, table, targets, 4)
        graph.capture_end()
    side.synchronize()
    x.copy_(x.flip(0))
    targets.copy_(targets.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    check(found, x.double() @ table.double().t(), targets, 4)
    del graph


def test_refusals():
    from pagedserve_b200.kernels.ops import KernelError

    ops = ops_for()
    logits, targets = torch.zeros(3, 50, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    for arguments in ((logits.double(), targets), (logits, targets.long()), (logits, targets[:2]), (logits, targets, 33), (logits, targets, -1),
                      (logits[:, :10], targets, 11), (logits.t(), targets), (logits[0], targets), (logits[:, :0], targets), (logits, targets.cpu()),
                      (torch.zeros(1, 50, device=DEV).expand(3, 50), targets)):
        with pytest.raises(KernelError):
            ops.token_logprobs(*arguments)
    table = torch.zeros(50, 8, device=DEV)
    for arguments in ((torch.zeros(3, 9, device=DEV), table, targets), (torch.zeros(3, 8, device=DEV).bfloat16(), table, targets),
                      (torch.zeros(3, 8, device=DEV), table, targets[:1]), (torch.zeros(3, 8, device=DEV), table.t(), targets)):
        with pytest.raises(KernelError):
            ops.head_logprobs(*arguments)
    good = ops.token_logprobs(logits, targets, 2)
    assert ops.token_logprobs(logits, targets, 2, results=good) is good
    for change in (dict(logprob=good.logprob[:2]), dict(entropy=good.entropy.double()), dict(top_logprobs=good.top_logprobs[:, :1]),
                   dict(top_ids=good.top_ids.long()), dict(top_ids=good.top_ids.t().contiguous().t()), dict(logprob=good.logprob.cpu())):
        with pytest.raises(KernelError):
            ops.token_logprobs(logits, targets, 2, results=good._replace(**change))
    with pytest.raises(KernelError):
        ops.token_logprobs(logits, targets.long(), 2, results=good)
    empty = ops.token_logprobs(logits[:0], targets[:0], 5)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 5)
    assert ops.head_logprobs(torch.zeros(0, 8, device=DEV), table, targets[:0]).entropy.shape == (0,)
