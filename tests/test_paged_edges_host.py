"""The serving operators without a GPU at the ends of their ranges: what the C
entries refuse, and the arithmetic of splits, record slots and page pools."""

import ctypes
import shutil
import subprocess
from pathlib import Path

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


# ---------------------------------------------------------------------------
# splits of long sequences
# ---------------------------------------------------------------------------
CSRC = Path(__file__).resolve().parents[1] / "dracort_b200" / "csrc"
LONGEST = 0x7FFF0000


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    """paged_split.h as the host's compiler sees it."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("needs a C++ compiler")
    d = tmp_path_factory.mktemp("split")
    (d / "s.cpp").write_text('#include "paged_split.h"\nextern "C" {\n'
                             "int count(int kend, int ck) { return draco::split_count(kend, ck); }\n"
                             "int end(int kbeg, int kend, int ck) { return draco::split_end(kbeg, kend, ck); }\n}\n")
    subprocess.run([gxx, "-O1", "-ftrapv", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "s.so"), str(d / "s.cpp")],
                   check=True)
    return ctypes.CDLL(str(d / "s.so"))


@pytest.mark.parametrize("kend", [1, 63, 64, 65, 9001, 1430000000, 1431655765, 1 << 30, LONGEST - 1, LONGEST])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 32, 63, 64])
def test_splits_cover_every_key_once(split, kend, n):
    for step in (1, 64, 128):  # what the kernels round a split's keys up to
        ck = ((kend + n - 1) // n + step - 1) // step * step
        count = split.count(kend, ck)
        assert count == -(-kend // ck) <= n
        ends = [split.end(s * ck, kend, ck) for s in range(count)]
        assert ends == [min(kend, (s + 1) * ck) for s in range(count)] and ends[-1] == kend


def test_a_sequence_of_no_keys_has_one_empty_split(split):
    assert split.count(0, 64) == 1 and split.end(0, 0, 64) == 0
