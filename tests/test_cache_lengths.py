"""Lengths and offsets in device memory that hold anything: the kernels' own arithmetic on them (csrc/lengths.hpp), in
constant expressions of the host's compiler, which accepts no overflow in one, and the kernels on a GPU."""

from __future__ import annotations

import itertools
import subprocess
from pathlib import Path

import pytest
import torch
from paged_oracle import Problem, attend, check_attention, quantise, sees

from ako_b200 import kv_cache_write_cuda_sm100, paged_attention_cuda_sm100

CSRC = Path(__file__).resolve().parent.parent / "ako_b200" / "csrc"
MIN, MAX = -(1 << 31), (1 << 31) - 1
ENDS = [MIN, MIN + 1, MIN + 300, -9, -1, 0, 1, 299, 300, 301, MAX - 1, MAX]


def compiles(tmp_path, lines) -> None:
    """The static assertions `lines` hold, and evaluating them overflows nowhere."""
    src = tmp_path / "lengths.cpp"
    literal = "constexpr int low = -2147483647 - 1;\n"
    src.write_text('#include "lengths.hpp"\nusing namespace ako_b200;\n' + literal + "\n".join(lines) + "\n")
    got = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsyntax-only", f"-I{CSRC}", str(src)],
                         capture_output=True, text=True)
    assert got.returncode == 0, got.stderr[:2000]


def text(x: int) -> str:
    return "low" if x == MIN else str(x)


def test_rows_of_any_two_offsets(tmp_path) -> None:
    lines = []
    for begin, end, tokens in itertools.product(ENDS, ENDS, (0, 1, 300, MAX)):
        first, last = (min(max(x, 0), tokens) for x in (begin, end))
        call = f"row_range({text(begin)}, {text(end)}, {text(tokens)})"
        lines.append(f"static_assert({call}.first == {first} && {call}.n == {max(last - first, 0)}, \"\");")
    compiles(tmp_path, lines)


def test_positions_of_any_length(tmp_path) -> None:
    lines = []
    for kv, n, held in itertools.product(ENDS, (1, 2, 300, MAX), (0, 1, 160, MAX - 4096)):
        for at in {0, n // 2, n - 1}:
            p = max(kv, 0) - n + at
            lines.append(f"static_assert(new_position({text(kv)}, {n}, {at}, {held}) == {p if 0 <= p < held else -1}, \"\");")
    compiles(tmp_path, lines)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
def test_tokens_past_the_table_take_no_earlier_place(cuda_device, quantised) -> None:
    """Tables of four pages of 8: lengths that end at the table's end, past it by fewer tokens than are new, by as
    many, and by far."""
    for ragged in (False, True):
        p = Problem(torch.bfloat16, quantised, 2, 2, 64, 8, [(4, 32)] * 5, ragged, 5, cuda_device)
        lens = [32, 34, 36, 1000, MAX]
        p.kv_lens = torch.tensor(lens, dtype=torch.int32)
        before = p.caches["k"].cpu().clone()
        kv_cache_write_cuda_sm100(p.k_new.to(cuda_device), p.v_new.to(cuda_device), p.kv(), p.batch())
        after = p.caches["k"].cpu()
        for b, n in enumerate(lens):
            for j in range(32):
                at = int(p.table[b, j // 8]), slice(None), j % 8
                i = j - (n - 4)
                if 0 <= i < 4:
                    new = p.rows(p.k_new, b)[i]
                    if quantised:
                        new = quantise(new)[0]
                    assert torch.equal(after[at].double(), new.double())
                else:
                    assert torch.equal(after.view(torch.uint8)[at], before.view(torch.uint8)[at])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 300], ids=["few", "many"])
def test_offsets_far_outside_the_tokens(cuda_device, new) -> None:
    """An odd group of heads (5 to a kv head). Sequences whose offsets run backwards or far past either end own the
    rows that lie between them and no others."""
    p = Problem(torch.bfloat16, False, 10, 2, 64, 16, [(new, new + 30), (new, new + 30), (new, new + 30)], True, 31,
                cuda_device)
    check_attention(p, paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch()))
    # Which keys a CTA takes, and with it the order of the fp32 sums, goes by all sequences' lengths: the last
    # sequence's rows are held to the bound of such sums and not to the bits of a call with other lengths.
    owned = slice(2 * new, 3 * new)
    want, bound = attend(p.q[owned], p.k[2], p.v[2], p.v_scale[2], sees(new, new + 30, 0, 0), 64**-0.5, p.dtype, False)
    for cu in ([new, MIN, 2 * new, 3 * new], [MAX, MIN, 2 * new, MAX], [MIN + new, MIN, 2 * new, MAX - 1]):
        # the second sequence holds rows 0 .. 2 * new - 1 where its begin is below 0
        p.cu = torch.tensor(cu, dtype=torch.int32)
        out = torch.full((3 * new + 2, 10, 64), 9.0, dtype=torch.bfloat16, device=cuda_device)
        q = torch.cat([p.q.to(cuda_device), torch.zeros(2, 10, 64, dtype=torch.bfloat16, device=cuda_device)])
        if cu[3] > 3 * new:  # the last sequence then owns the two rows behind the others'
            q, out = q[:3 * new], out[:3 * new]
        paged_attention_cuda_sm100(q, p.kv(), p.batch(), out=out)
        assert bool(((out[owned].double().cpu() - want).abs() <= bound).all())
        assert bool(torch.isfinite(out).all()) and bool((out[3 * new:] == 9).all())
        before = {name: p.caches[name].clone() for name in ("k", "v")}
        kv_cache_write_cuda_sm100(p.k_new.to(cuda_device), p.v_new.to(cuda_device), p.kv(), p.batch())
        pages = [int(x) for x in p.table[0]]  # of the first sequence, which has no rows
        for name in ("k", "v"):
            assert torch.equal(p.caches[name][pages].view(torch.int16), before[name][pages].view(torch.int16))
            p.caches[name].copy_(before[name])
