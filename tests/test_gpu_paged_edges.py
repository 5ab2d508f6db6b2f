"""The serving operators over the paged cache at the ends of their ranges."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

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
