"""Log probabilities and entropies of rows where one token has nearly all the mass, to a relative bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def tail64(x, t):
    """Of rows x (R, V) whose largest logit is x[r, t[r]]: log probability of t, entropy, and how
    far below the maximum the terms of both sums lie, weighted by their size."""
    lp, ent, far = [], [], []
    for r in range(x.shape[0]):      # a row at a time: 64 bits of all of them would be large
        d = x[r].double() - x[r, t[r]].double()
        e = d.exp()
        e[t[r]] = 0.0                # the 1 that would hide the others
        tail = e.sum()
        d = d.clamp_min(-1e5)
        w = (e * d).sum()
        lp.append(-torch.log1p(tail))
        ent.append(torch.log1p(tail) - w / (1 + tail))
        far.append(torch.maximum(-w / tail, (e * d * d).sum() / -w))
    return torch.stack(lp), torch.stack(ent), torch.stack(far)


def relative_bound(far, V):
    """A term e^d is off by what 32 bits lose of d (its subtraction, its product with log2 e and that
    constant: 2.5 roundings of 2^-24 |d|) and by 2^-22 from the exponential; it passes through
    at most V / 64 + 64 sums (a warp's 32 lanes add two at a time; longer rows have four warps at
    least); the logarithm and the quotient add a few units more."""
    sums = V / (64 if V <= 8448 else 256) + 64
    return 2.5 * 2.0 ** -24 * far + 2.0 ** -21 + sums * 2.0 ** -24


# rows of few vectors, rows of a warp, of a CTA (once, and in several tiles), of clusters
SHAPES = [(3, 31), (40, 500), (900, 350), (900, 6563), (600, 9001), (300, 20011), (600, 50001), (80, 30001), (1, 6563),
          (1, 151000), (1, 1048576)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("R,V", SHAPES)
def test_likely_tokens_keep_their_digits(dtype, R, V):
    from yapd_b200.logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(V + R)
    for pad in (0, 1, 5):
        base = torch.randn(R, V + pad, generator=g, device="cuda") * 2
        x = base.to(TYPES[dtype])[:, pad:]          # rows that begin anywhere in a vector
        t = torch.randint(0, V, (R,), generator=g, device="cuda")
        t[::7], t[1::7], t[2::7] = 0, V - 1, min(V - 1, 3)
        lead = torch.tensor([5.0, 10.0, 20.0, 30.0], device="cuda").repeat(-(-R // 4))[:R]
        if R == 1:
            lead[:] = (20.0, 30.0, 10.0)[(0, 1, 5).index(pad)]
        rows = torch.arange(R, device="cuda")
        x[rows, t] = (x.float().amax(1) + lead).to(x.dtype)
        lp, ent, far = tail64(x, t)
        bound = relative_bound(far, V)
        for top_n in (0, 3):
            got = token_logprobs(x, t, top_n=top_n)
            for have, want in ((got.logprob, lp), (got.entropy, ent)) + (((got.top_logprobs[:, 0], lp),) if top_n else ()):
                err = ((have.double() - want) / want).abs()
                assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_ties_and_lone_tokens(dtype):
    """Equal largest logits count as often as they are there; a token alone has probability 1."""
    from yapd_b200.logprobs import token_logprobs
    import math
    for V in (2, 40, 3001, 9001, 100003):
        x = torch.full((6, V), -math.inf, dtype=TYPES[dtype], device="cuda")
        x[0, V // 2] = 2.0
        x[1, 0] = x[1, V - 1] = -7.0
        x[2] = 3.0
        x[3, V - 1] = 1.0
        x[4, : max(2, V // 2)] = 0.0
        x[5, ::2] = -0.0
        x[5, 1] = 0.0
        n = [1, 2, V, 1, max(2, V // 2), (V + 1) // 2 + 1]
        t = torch.tensor([V // 2, 0, V - 1, V - 1, 1, 0], device="cuda")
        got = token_logprobs(x, t, top_n=1)
        want = -torch.tensor(n, dtype=torch.float64).log()
        for have, sign in ((got.logprob, 1), (got.top_logprobs[:, 0], 1), (got.entropy, -1)):
            err = (have.cpu().double() - sign * want).abs()
            assert bool((err <= (V / 64 + 64) * 2.0 ** -24 * want.abs()).all()), (V, err)


def test_more_rows_than_32_bits_count_are_refused():
    """2^32 + 3 rows are not 3."""
    from yapd_b200.logprobs import token_logprobs
    x = torch.zeros(1, 1, device="cuda").expand(2 ** 32 + 3, 1)
    with pytest.raises(ValueError):
        token_logprobs(x)
