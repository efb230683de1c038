"""Log probabilities of rows whose parts hold several batches (4096 logits each): two batches in turn, even and odd counts and ragged ends; a larger maximum, ties, masks
and NaN that meet what an earlier batch has left; the bounds behind batch 1, 2, 4, ...; 64 parts joined.  Against 64 bits, as every row of test_ops_gpu."""
import math
from importlib import import_module

import numpy as np
import pytest
import torch

import __graft_entry__ as ge
from test_ops_gpu import DEV, NAMES, check_rows, rng

pytestmark = pytest.mark.gpu
BATCH = 4096


@pytest.fixture(scope="module")
def ops(pkg):
    return import_module(ge.PKG_NAME + ".ops")


def rows_of(vocab, dtype, seed):
    """Rows by name -> float32 [vocab]; all within what the type holds without rounding two different logits of a ramp to one where that matters."""
    r = rng(seed)
    low = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}[dtype]
    noise = lambda: (r.standard_normal(vocab) * 3).astype(np.float32)
    step = np.arange(vocab) // 7          # runs of equal logits, across every border of vectors, lanes and batches
    last = (vocab - 1) // BATCH * BATCH          # the last batch's first token of a row that is one part
    rows = {"noise": noise()}
    rows["rising"] = (step * (80.0 / max(1, step[-1]))).astype(np.float32)          # the largest logit is always the next one
    rows["falling"] = -rows["rising"]
    rows["steep"] = (step * (4000.0 / max(1, step[-1]))).astype(np.float32)
    rows["batches rise"] = noise() + np.float32(9) * (np.arange(vocab) // BATCH)
    rows["batches fall"] = noise() - np.float32(9) * (np.arange(vocab) // BATCH)
    rows["few values"] = r.integers(-1, 2, vocab).astype(np.float32)
    rows["equal"] = np.full(vocab, 2.5, np.float32)
    rows["equal, one more at the end"] = np.full(vocab, 2.5, np.float32); rows["equal, one more at the end"][-1] = 3
    x = noise() * 0.1; x[BATCH - 3:BATCH + 3] = 5; x[last:last + 2] = 5; rows["ties across a border"] = x
    x = noise() * 0.1; x[::BATCH // 4] = 6; rows["ties in every batch"] = x
    x = np.full(vocab, -np.inf, np.float32); x[last:] = noise()[last:]; rows["masked up to the last batch"] = x
    x = np.full(vocab, -np.inf, np.float32); x[:40] = noise()[:40]; rows["masked behind the first vectors"] = x
    x = noise(); x[BATCH:2 * BATCH] = -np.inf; rows["a masked batch"] = x
    x = np.full(vocab, -np.inf, np.float32); x[r.random(vocab) < 0.001] = 1.25; x[-1] = 1.25; rows["few left, all equal"] = x
    rows["all masked"] = np.full(vocab, -np.inf, np.float32)
    x = np.full(vocab, low, np.float32); x[last // 2] = -2; x[-1] = -2; rows["masked with the lowest value"] = x
    x = noise(); x[5] = np.nan; rows["NaN at the start"] = x
    x = noise(); x[-1] = np.nan; rows["NaN at the end"] = x
    x = np.full(vocab, -np.inf, np.float32); x[3] = np.nan; x[-2] = 4; rows["NaN in front of the only token"] = x
    x = noise(); x[last] = np.inf; rows["+inf in the last batch"] = x
    x = noise(); x[0] = np.inf; rows["+inf first"] = x
    x = noise(); x[vocab // 2] += 40; rows["certain in the middle"] = x
    x = noise() * 0.01 - 3000; rows["far from zero"] = x
    return rows


def check(ops, rows, vocab, dtype, top, sample, pad=0, first=0):
    special = rows_of(vocab, dtype, 100 * vocab % 99991 + top)
    names = list(special)
    r = rng(vocab + rows)
    wide = torch.randn(rows, first + vocab + pad, generator=torch.Generator(device=DEV).manual_seed(vocab), device=DEV) * 3
    at = [int(i) for i in r.permutation(rows)[:len(names)]] if rows > len(names) else list(range(rows))
    for i, name in zip(at, names):
        wide[i, first:first + vocab] = torch.from_numpy(special[name]).to(DEV)
    x = wide.to(NAMES[dtype])[:, first:first + vocab]
    last = (vocab - 1) // BATCH * BATCH
    t = torch.from_numpy(r.integers(0, vocab, rows).astype(np.int32)).to(DEV)
    places = [0, 3, BATCH - 1, BATCH, BATCH + 1, vocab // 2, last, last + 1, vocab - 1, vocab - 2, -1]
    for j, i in enumerate(at):
        t[i] = min(places[(j + top) % len(places)], vocab - 1)
    got = ops.token_logprobs(x, t, top)
    some = at + [int(i) for i in r.integers(0, rows, sample)]
    pick = torch.tensor(some, device=DEV)
    check_rows(type(got)(*(v[pick] if v is not None else None for v in got)), x[pick], t[pick], top)
    # the same rows with every place of the target, once per batch border
    for place in places[:-1]:
        t2 = torch.full((rows,), min(place, vocab - 1), dtype=torch.int32, device=DEV)
        other = ops.token_logprobs(x, t2, 0)
        assert torch.equal(other.entropy.nan_to_num(7e30), got.entropy.nan_to_num(7e30))
        check_rows(type(other)(*(v[pick] if v is not None else None for v in other)), x[pick], t2[pick], 0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(700, 5003, 20), (700, 8192, 1), (700, 8193, 64), (700, 12300, 64), (700, 16384, 5), (700, 20479, 1), (650, 32064, 20)])
def test_a_row_is_one_part(ops, dtype, rows, vocab, top):
    """2, 2, 3, 4, 4, 5 and 8 batches, whole and ragged."""
    check(ops, rows, vocab, dtype, top, 4)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top,pad,first", [(500, 40000, 20, 0, 0), (500, 40000, 64, 7, 3), (300, 50257, 1, 1, 1), (40, 300000, 33, 0, 0), (1300, 9001, 64, 5, 2)])
def test_rows_of_several_parts_and_odd_strides(ops, dtype, rows, vocab, top, pad, first):
    """Two parts of 5 batches, four of 4, 32 of 3; rows that start anywhere in a vector."""
    check(ops, rows, vocab, dtype, top, 2, pad, first)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [258049, 262144, 300001, 1100003])
def test_as_many_parts_as_are_joined(ops, dtype, vocab):
    """64 parts of a batch, then 37 and 54 of two and five; every kind of row by itself and as one of three."""
    special = rows_of(vocab, dtype, vocab)
    for n in (1, 3):
        for i in range(0, len(special), 5 if n == 1 else 3):
            names = list(special)[i:i + n]
            x = torch.from_numpy(np.stack([special[k] for k in names])).to(NAMES[dtype]).to(DEV)
            t = torch.tensor([vocab - 1, 4096, 0][:len(names)], dtype=torch.int32, device=DEV)
            for top in (64, 3):
                check_rows(ops.token_logprobs(x, t, top), x, t, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_token_in_every_place(ops, dtype):
    """One row, the target at every id around the borders of vectors, wavefronts and batches: logprob and rank of a falling and of an all-equal row are their ids'."""
    vocab, rows = 12301, 2600
    for kind in ("equal", "falling"):
        row = torch.zeros(vocab) if kind == "equal" else -torch.arange(vocab, dtype=torch.float32) * 2.0 ** -7
        x = row.to(NAMES[dtype]).to(DEV).repeat(rows, 1)
        t = torch.from_numpy(np.concatenate([np.arange(0, 700), np.arange(3900, 4300), np.arange(8000, 8400), np.arange(11201, 12301)]).astype(np.int32)).to(DEV)
        assert t.numel() == rows
        got = ops.token_logprobs(x, t, 64)
        assert torch.equal(got.rank.long(), t.long() + 1)          # (equal logits: lower id first; rounded ones are equal in runs)
        assert torch.equal(got.top_ids, torch.arange(64, dtype=torch.int32, device=DEV).repeat(rows, 1))
        if kind == "equal":
            assert ((got.logprob + math.log(vocab)).abs() < 1e-5).all() and ((got.entropy - math.log(vocab)).abs() < 1e-5).all()
