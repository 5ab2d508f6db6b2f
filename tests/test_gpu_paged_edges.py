"""The serving operators over the paged cache at the ends of their ranges."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import test_gpu_paged as T  # noqa: E402
from dracort_b200 import paged_ops as P  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF16 = torch.float32, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("tokens,dtype", [(1, F32), (1, BF16), (256, BF16)])
def test_the_longest_sequence(tokens, dtype):
    """0x7FFF0000 positions on two pages that the table repeats: values of 1 in the first nine tenths and 2 behind
    them, all scores equal.  The sums are whole numbers that fp32 holds; 2^-8 is the output's rounding."""
    page, hd, length = 1024, 32, 0x7FFF0000
    k, v = P.kv_cache("bf16", 2, 1, page, hd, DEV)
    v[0], v[1] = 1.0, 2.0
    pages = length // page
    table = torch.zeros((1, pages), dtype=torch.int32, device=DEV)
    table[:, pages * 9 // 10:] = 1
    want = 1 + (pages - pages * 9 // 10) / pages
    out = P.attention_paged(torch.zeros(tokens, 1, hd, dtype=dtype, device=DEV), k, v, table, i32([0, tokens]),
                            i32([length]), max_q=tokens, max_kv=length)
    assert P.attention_paged_status() == 0
    assert float((out.double() - want).abs().max()) <= want * 2.0 ** -8


@pytest.mark.parametrize("heads,kv", [(8, 8), (8, 2), (6, 1), (40, 2)])
@pytest.mark.parametrize("cache", ["bf16", "q8_0"])
def test_chunks_among_many_steps(cache, heads, kv):
    """Chunks that are split, at several places among 90 sequences of a token or none, some at the least length that
    the long chunks' kernel takes; run again, the same numbers."""
    least = 64 // (heads // kv) + 1
    new = [1, 0, 1, 1] * 22 + [1, 1]
    new[0], new[30], new[31], new[60], new[89] = least, 290, least, least - 1, 150
    past = [(s * 131) % 700 for s in range(90)]
    past[0], past[30], past[31], past[89] = 3000, 2500, 4000, 2000
    b = T.batch(new, past, heads, kv, 64, 64, cache, BF16, seed=41)
    out = torch.full_like(b[0], float("nan"))
    P.attention_paged(*b, max_q=290, max_kv=4000 + least, out=out)
    T.check(*b, out)
    for _ in range(3):
        assert torch.equal(P.attention_paged(*b, max_q=290, max_kv=4000 + least), out)
