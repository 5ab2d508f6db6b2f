"""The serving operators without a GPU at the ends of their ranges: what the C
entries refuse, and the arithmetic of splits, record slots and page pools."""

import ctypes
import random
import shutil
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from dracort_b200 import _native as N
from dracort_b200 import paged_ops as P

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
                             "int end(int kbeg, int kend, int ck) { return draco::split_end(kbeg, kend, ck); }\n"
                             "long long place(int start, int row0, int group, int R, int from) {\n"
                             "  return draco::record_place(start, row0, group, R, from); }\n"
                             "long long places(int n, int group, int R, int from) {\n"
                             "  return draco::record_places(n, group, R, from); }\n}\n")
    subprocess.run([gxx, "-O1", "-ftrapv", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "s.so"), str(d / "s.cpp")],
                   check=True)
    so = ctypes.CDLL(str(d / "s.so"))
    so.place.restype = so.places.restype = ctypes.c_longlong
    return so


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


# ---------------------------------------------------------------------------
# partial results of long chunks beside many short sequences
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 20, 64, 65, 128])
def test_long_chunks_have_places_of_their_own(split, group):
    rng = random.Random(group)
    rows, frm = 2 * group * (128 // group), 64 // group + 1
    for _ in range(200):
        new = [rng.choice([0, 1, 1, frm - 1, frm, frm, frm + 1, rng.randint(1, 3 * rows // group + 1)])
               for _ in range(rng.randint(1, 60))]
        n, start, seen = sum(new) + rng.choice([0, 0, 5]), 0, []
        for m in new:
            if m >= frm:
                seen += [split.place(start, r, group, rows, frm) for r in range(0, m * group, rows)]
            start += m
        assert len(set(seen)) == len(seen)
        assert all(0 <= p < split.places(n, group, rows, frm) for p in seen)
    # the places of any token count stay in range, at the largest ones too
    n = 0x7FFF0000 // group
    last = (frm * group - 1) // rows * rows
    assert split.place(n - frm, last, group, rows, frm) < split.places(n, group, rows, frm)


@pytest.mark.parametrize("heads,kv,head_dim", [(8, 8, 128), (32, 8, 128), (32, 32, 64), (6, 1, 96), (64, 1, 128)])
def test_workspace_of_many_steps_beside_a_chunk(heads, kv, head_dim):
    """What a batch of steps and one or several chunks takes is bounded by the tokens, not by the sequences."""
    for steps in (0, 1, 10, 64, 200, 1000):
        for chunks, size in ((1, 100), (1, 512), (3, 700), (1, 4000)):
            c = N.KvCache(type=N.KV_BF16, kv_heads=kv, head_dim=head_dim, page_size=64, n_pages=8, n_seqs=steps + chunks,
                          max_pages=256, table_stride=256, k=PTR, v=PTR, block_table=PTR)
            need = lib.draco_attention_paged_workspace_bytes(c, steps + chunks * size, heads, size, 8000, N.DTYPE_BF16)
            assert N.PAGED_WORKSPACE_HEAD <= need < 200 << 20, (steps, chunks, size, need)


def test_status_needs_a_place_for_it():
    assert lib.draco_attention_paged_status(0, None) == N.DRACO_ERR_ARG


# ---------------------------------------------------------------------------
# tensors on another device than the current one (fakes: one device is enough)
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("capturing", [None, 0, 1])
def test_attention_on_another_device_than_the_current_one(capturing, monkeypatch):
    """Device 0 is current, the tensors are on device 1: the capture that counts is device 1's, sizes are asked, the
    workspace is made and the call is enqueued with device 1 current."""
    current, seen = [0], []

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            self.before, current[0] = current[0], self.d

        def __exit__(self, *e):
            current[0] = self.before

    class Lib:
        def attention_paged(self, *args):
            seen.append(("call", current[0], args[-1]))
            return N.DRACO_ERR_WORKSPACE if sum(s[0] == "call" for s in seen) == 1 and capturing != 1 else 0

        def workspace_bytes(self, *args):
            seen.append(("size", current[0]))
            return 1 << 14

    cache = SimpleNamespace(get_device=lambda: 1, new_empty=lambda n, dtype: (
        seen.append(("workspace", current[0], n)) or torch.empty(n, dtype=dtype)))
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == capturing)
    for name, fake in (("_current_device", lambda: current[0]), ("_current_stream", lambda d: 100 + d),
                       ("_cache_struct", lambda *a: (b"", 2, 1, 64)), ("_rows", lambda *a: 64),
                       ("_vector", lambda *a: 0), ("_lib", Lib), ("_workspaces", {})):
        monkeypatch.setattr(P, name, fake)
    P.attention_paged(torch.zeros(1, 2, 32), cache, None, None, None, None)
    assert current == [0] and {s[1] for s in seen} == {1}
    assert [s for s in seen if s[0] == "call"][-1] == ("call", 1, 101)
    assert [s[2] for s in seen if s[0] == "workspace"] == [1 << 14 if capturing == 1 else 1 << 20]
    assert list(P._workspaces) == ([] if capturing == 1 else [(1, 101)])
