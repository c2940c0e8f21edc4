"""Wide rows that hold more candidates for their likeliest classes than the kernel's list, and take them one maximum after
another instead: rows of distinct values, not of equal ones alone, in every form of the kernel.  ``candidates`` counts what the
list would have to hold, from the columns that the kernel's threads look at."""
import sys

import pytest
import torch

from test_labels import check

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LIST, PARTS, TOP = 2048, 128, 32


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def form(rows, classes, dtype):
    """(columns of a split, threads of its workgroup, values of a vector)."""
    size = torch.finfo(dtype).bits // 8
    v = 16 // size
    need = -(-classes // (1024 * 8 * v))
    want = max(need, min(64, max(1, 512 // rows), max(1, classes // 4096)))
    cols = -(--(-classes // want) // v) * v
    return cols, 256 if -(-cols // v) <= 2048 else 1024, v


def part_of(rows, classes, dtype):
    """The split and the part of each column."""
    cols, threads, v = form(rows, classes, dtype)
    col = torch.arange(classes)
    return col // cols, col % cols // v % threads // (threads // PARTS)


def candidates(row, rows, dtype, top=TOP):
    """Most values that any split of the row has at or above its bound, the top-th largest of its parts' maxima."""
    split, part = part_of(rows, row.numel(), dtype)
    most = 0
    for s in range(int(split.max()) + 1):
        x, p = row[split == s].double(), part[split == s]
        maxima = torch.full((PARTS,), -float("inf"), dtype=torch.float64).scatter_reduce(0, p, x, "amax")
        most = max(most, int((x >= maxima.sort(descending=True).values[top - 1]).sum()))
    return most


def distinct(rows, classes, seed):
    """Rows of distinct values in [0, 1), as far as the type tells them apart."""
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.randperm(classes, generator=g) for _ in range(rows)]).float() / classes


def test_the_forms_that_are_tested():
    assert form(513, 20000, F32) == (20000, 1024, 4) and form(513, 20000, BF16) == (20000, 1024, 8)
    assert form(513, 16000, BF16) == (16000, 256, 8) and form(513, 8000, F32) == (8000, 256, 4)
    assert form(513, 60000, F32) == (30000, 1024, 4) and form(100, 60000, F32) == (12000, 1024, 4)
    assert form(1, 100000, F32) == (4168, 256, 4) and form(513, 40000, F16) == (40000, 1024, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype", [(513, 20000, F32), (513, 20000, BF16), (513, 40000, F16), (513, 16000, BF16),
                                                (513, 60000, F32), (100, 60000, F32)])
def test_large_values_in_few_parts(gpu, rows, classes, dtype):
    """31 parts of a split hold all the large values, so the bound, the 32nd part's maximum, lies below every one of them."""
    say("crowd", rows, classes, dtype)
    z = distinct(rows, classes, 1)
    split, part = part_of(rows, classes, dtype)
    z[0] += 5.0 * (part < 31)
    z[1] += 5.0 * (part >= 97)
    z[2] += 5.0 * ((part * 37) % PARTS < 31)
    z[3] += 5.0 * ((part < 31) & (split == split.max()))
    z[4] = -z[0]
    z = z.to(dtype)
    for r in (0, 1, 2, 3):
        assert candidates(z[r], rows, dtype) > LIST, r
    y = torch.randint(0, classes, (rows,), generator=torch.Generator().manual_seed(2))
    check(gpu, z, y, TOP, ("crowd", rows, classes, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype", [(513, 8000, F32), (513, 20000, F32), (1, 100000, F32), (1, 100000, BF16), (3, 50000, F16),
                                                (100, 60000, F32), (513, 2500, BF16)])
def test_masked_rows_with_values_in_few_parts(gpu, rows, classes, dtype):
    """-inf everywhere but in some columns of fewer parts than classes asked for: the bound is -inf, and all columns reach it."""
    say("masked crowd", rows, classes, dtype)
    z = distinct(rows, classes, 3)
    split, part = part_of(rows, classes, dtype)
    picks = [part < 31, part >= 120, (part == 64) | (part == 65), (part < 31) & (split == 0)]
    for r in range(min(rows, len(picks))):
        z[r, ~picks[r]] = -float("inf")
    z = z.to(dtype)
    for r in range(min(rows, len(picks))):
        assert candidates(z[r], rows, dtype) > LIST, r
    y = torch.stack([(z[r] > -float("inf")).nonzero()[0, 0] for r in range(rows)])
    check(gpu, z, y, TOP, ("masked crowd", rows, classes, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [LIST - 1, LIST, LIST + 1])
def test_a_list_that_is_just_full(gpu, count):
    """As many candidates as the list holds, one fewer and one more."""
    rows, classes = 513, 20000
    say("full list", count)
    z = distinct(rows, classes, 4)
    _, part = part_of(rows, classes, F32)
    at = (part < 31).nonzero()[:, 0]
    z[0, at[torch.randperm(at.numel(), generator=torch.Generator().manual_seed(5))[:count - 1]]] += 5.0
    rest = part >= 31
    z[0, at] = torch.where(z[0, at] < 2.0, z[0, at] * 0.5 - 1.0, z[0, at])      # the others there lie below the bound
    assert int((z[0, rest] >= z[0, rest].max()).sum()) == 1 and candidates(z[0], rows, F32) == count
    y = torch.randint(0, classes, (rows,), generator=torch.Generator().manual_seed(6))
    check(gpu, z, y, TOP, ("full list", count))
