"""The serving operators without a GPU at the ends of their ranges: what the C
entries refuse, and the arithmetic of splits, record slots and page pools."""

import pytest

from dracort_b200 import _native as N

PTR = 1 << 20  # an aligned address; every call below returns before it would be read

lib = N.load()


def verify_at(temperature, **kw):
    f = dict(logits=PTR, draft_probs=None, row_start=PTR, drafts=PTR, accept_u=PTR, sample_u=PTR, accepted=PTR,
             tokens=PTR, ld_logits=100, ld_probs=0, ld_tokens=4, temperature=-1.0, dtype=N.DTYPE_F32, n=5, n_seqs=2,
             vocab=100, max_rows=4)
    f.update(kw)
    return lib.draco_verify_drafts_at(N.VerifyArgs(**f), temperature, None)


@pytest.mark.parametrize("temperature", [-0.5, 1e-46, 9.9e-31, 1.1e30, float("nan"), float("inf")])
def test_temperatures_of_64_bits_that_are_refused(temperature):
    assert verify_at(temperature) == N.DRACO_ERR_ARG
    assert "temperature" in N.last_error()


def test_verification_at_a_temperature_checks_what_the_fp32_form_checks():
    assert verify_at(0.8, n_seqs=0) == N.DRACO_OK  # (the structure's own temperature is not read)
    assert verify_at(0.8, sample_u=None) == N.DRACO_ERR_ARG
    assert verify_at(0.8, vocab=0) == N.DRACO_ERR_SHAPE
    assert verify_at(0.8, logits=PTR + 2) == N.DRACO_ERR_ALIGN
    assert lib.draco_verify_drafts_at(None, 1.0, None) == N.DRACO_ERR_ARG
