"""Token log probabilities, entropy and alternatives against 64-bit formulas."""
import math

import pytest
import torch

from tests.serve_util import logprobs64

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(x, targets, top_n):
    """Errors that 32-bit arithmetic explains: x - max and its sum with -ln z are rounded to 24 bits;
    exp is off by 2^-22 relative, its argument by 2^-24 |x - max|; a sum of V terms over at least 64
    threads loses (V / 64 + 16) 2^-24 of the sum of the terms' sizes."""
    from yapd_b200.logprobs import token_logprobs
    got = token_logprobs(x, targets.to(x.device), top_n=top_n)
    own, entropy, top, ids, spread = logprobs64(x.cpu(), targets.cpu().long(), top_n)
    V = x.shape[1]
    unit = (V / 64 + 64) * 2.0 ** -24 + 2.0 ** -20
    for have, want, size in ((got.logprob, own, own.abs()), (got.entropy, entropy, 2 * spread),
                             (got.top_logprobs, top, top.abs()) if top_n else (got.entropy, entropy, 2 * spread)):
        have = have.cpu().double()
        assert torch.equal(have.isnan(), want.isnan())
        assert torch.equal(have == -math.inf, want == -math.inf)
        fin = want.isfinite()
        err, tol = (have - want).abs()[fin], (unit * (1 + size))[fin]
        assert bool((err <= tol).all()), float((err / tol).max())
    if top_n:
        assert torch.equal(got.top_ids.cpu().long(), ids)
    return got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("R,V,top_n", [(1, 1, 1), (3, 2, 5), (2, 7, 32), (5, 33, 0), (4, 513, 20), (3, 6563, 5),
                                       (9, 8194, 8), (2, 50001, 32), (1, 151000, 20), (1, 1048576, 1), (700, 65, 3)])
def test_logprobs(dtype, R, V, top_n):
    g = torch.Generator().manual_seed(V)
    x = (2 * torch.randn(R, V, generator=g)).to(TYPES[dtype])
    targets = torch.randint(0, V, (R,), generator=g)
    check(x.cuda(), targets, top_n)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_with_masks_ties_and_nothing(dtype):
    V, inf, nan = 3000, float("inf"), float("nan")
    x = torch.randn(14, V, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype])
    x[0] = 0.0                              # all equal
    x[1] = -inf                             # nothing left
    x[2] = -inf
    x[2, 1234] = 5.0                        # one token left
    x[3, 17] = nan
    x[4, V - 1] = inf
    x[5] = torch.finfo(x.dtype).min         # a mask of the type's lowest value everywhere but two
    x[5, 7], x[5, 99] = 3.0, 2.0
    x[6, ::3] = -inf
    x[7] = torch.finfo(x.dtype).min         # and everywhere
    x[8, ::2] = 7.0                         # half of the row ties for the first place
    x[9, 5::7], x[9, 6::7] = 0.0, -0.0      # zeros of both signs are equal
    x[9] = x[9].clamp_max(0)
    x[10] = -inf
    x[10, 20:25] = 1.0                      # fewer than asked for, all equal
    x[11, -40:] = 9.0
    x[12] = x[12].sort().values
    x[13, :] = torch.linspace(-60000.0, 60000.0, V).to(x.dtype)
    targets = torch.tensor([0, 5, 1234, 17, 3, 7, 0, 12, 1, 5, 24, V - 1, -1, V])
    for top_n in (1, 8, 32):
        check(x.cuda(), targets, top_n)


def test_strides_and_types_of_targets():
    base = torch.randn(40, 1009, generator=torch.Generator().manual_seed(2))
    for dt in TYPES.values():
        for lo, hi in ((0, 1000), (1, 1001), (3, 9), (5, 1009)):
            x = base.to(dt).cuda()[1:, lo:hi]                       # odd starts and row strides
            t = torch.arange(39, dtype=torch.int32) % (hi - lo)
            check(x, t, 4)
        check(base.to(dt).cuda().t(), torch.zeros(1009, dtype=torch.int64), 2)     # strided columns: a copy
        check(base.to(dt).cuda()[:1].expand(6, -1), torch.arange(6), 3)            # a broadcast row
    none = check(base[:0].cuda(), torch.zeros(0, dtype=torch.int64), 3)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 3)


def test_rows_past_32_bits_and_another_stream():
    from yapd_b200.logprobs import token_logprobs
    V, R = 65536, 65600                              # 2^32 elements and some more
    x = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(V, device="cuda").to(torch.bfloat16)
    x[-1, 777] = 30.0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t = torch.full((R,), 777, device="cuda")
        got = token_logprobs(x, t, top_n=1)
    torch.cuda.current_stream().wait_stream(side)
    assert int(got.top_ids[-1, 0]) == 777 and float(got.logprob[-1]) > -1e-6
    assert float((got.logprob[:-1] + math.log(V)).abs().max()) < 1e-4
    assert float((got.entropy[:-1] - math.log(V)).abs().max()) < 1e-4
    assert int(got.top_ids[:-1].abs().max()) == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V", [9, 31, 64, 200, 459, 767, 768, 1100])
def test_short_rows_with_many_alternatives(dtype, V):
    """Rows whose lanes hold a few tokens each, masks, ties and all."""
    g = torch.Generator().manual_seed(V)
    x = (2 * torch.randn(40, V, generator=g)).to(TYPES[dtype])
    x[1::4][torch.rand(10, V, generator=g) < 0.5] = float("-inf")
    x[2::4] = x[2::4].round()
    x[3::8] = x[3::8].sort(1).values
    x[:, V // 2] = 1.0
    for top_n in (9, 17, 32):
        check(x.cuda(), torch.randint(0, V, (40,), generator=g), top_n)
