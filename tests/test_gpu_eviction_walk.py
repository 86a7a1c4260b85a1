"""Eviction of rows that the in-place walk takes in several chunks and lists, in both block sizes of the kernel, with the sums in
shared memory and without: kept and equal tokens counted over chunks, lists that wait for the next chunk, places in earlier
chunks.  Exact: the bytes are those of the definition."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_paged_eviction import Pool

pytestmark = pytest.mark.gpu


class Long(Pool):
    """The same pool, its definition written for whole heads; planes of random bits."""

    def __init__(self, lens, layers=1, nh=1, hd=64, bs=16, seed=0, width=None, sums="random"):
        super().__init__(lens, layers, nh, 16, bs, torch.float16, seed, width=width, sums=sums)  # planes are made below
        g = torch.Generator().manual_seed(seed)
        self.keys, self.values = (torch.randint(-2**15, 2**15, (layers, self.pages, bs, nh, hd), generator=g, dtype=torch.int16).view(torch.float16)
                                  for _ in range(2))
        if sums == "few":  # half of them equal, the others below and above
            self.sums = torch.where(self.sums < 0.5, 0.5, self.sums.mul(8).floor())

    def evicted(self, rows, keep, sinks, recent):
        tables, lens, refs, keys, values, sums = self.state()
        keys, values = keys.view(torch.int16), values.view(torch.int16)
        for row in rows:
            n = int(lens[row])
            if n <= keep:
                continue
            held, written = -(-n // self.bs), -(-keep // self.bs)
            t = torch.arange(n)
            page, place = tables[row].long()[t // self.bs], t % self.bs
            for layer in range(self.layers):
                for h in range(self.nh):
                    x = sums[layer, row, h, :n].clone()
                    order = x[sinks:n - recent].nan_to_num(nan=-torch.inf, posinf=torch.inf, neginf=-torch.inf).sort(descending=True, stable=True).indices
                    stay = torch.zeros(n, dtype=torch.bool)
                    stay[:sinks] = True
                    stay[n - recent:] = True
                    stay[order[:keep - sinks - recent] + sinks] = True
                    stay = stay.nonzero()[:, 0]
                    assert len(stay) == keep
                    for plane in (keys, values):
                        plane[layer, page[:keep], place[:keep], h] = plane[layer, page[stay], place[stay], h]
                    sums[layer, row, h] = 0
                    sums[layer, row, h, :keep] = x[stay]
            refs[tables[row, written:held].long()] -= 1
            tables[row, written:held] = -1
            lens[row] = keep
        return [tables, lens, refs, keys.view(torch.float16), values.view(torch.float16), sums], 0


def test_the_two_definitions_agree():
    for sums in ("random", "ties"):
        p = Pool([200, 64, 65, 130], sums=sums)
        q = Long([200, 64, 65, 130], 2, 2, sums=sums)
        q.tables, q.refs, q.keys, q.values, q.sums = p.tables, p.refs, p.keys.view(torch.float16), p.values.view(torch.float16), p.sums
        for args in (([0, 2, 3], 40, 3, 9), ([0, 1, 2, 3], 64, 0, 0)):
            (a, left), (b, _) = p.evicted(*args), q.evicted(*args)
            assert left == 0
            for x, y in zip(a, b):
                assert torch.equal(x.view(torch.int16) if x.dtype.itemsize == 2 else x, y.view(torch.int16) if y.dtype.itemsize == 2 else y)


# A block of 512 threads: chunks of 4096 tokens, lists of 8192.
@pytest.mark.parametrize("sums", ["random", "ties", "few"])
@pytest.mark.parametrize("n", [4095, 4096, 4097, 8191, 8193, 12289, 20000])
def test_long_rows_of_few_heads(n, sums):
    for keep, sinks, recent in ((1000, 4, 100), (n // 2 + 1, 0, 0), (n - 1, 0, 0), (n - 3, 4097 if n > 8192 else 1, n // 3), (1, 0, 0)):
        Long([n, 70], nh=2, sums=sums).check([0, 1], keep, sinks, recent)


@pytest.mark.parametrize("hd,bs", [(128, 64), (256, 24)])
def test_long_rows_of_wide_heads(hd, bs):
    Long([9001, 4300], hd=hd, bs=bs, sums="ties").check([0, 1], 4200, 2, 30)


# More blocks than SMs, 256 threads: chunks of 2048 tokens, lists of 4096.
MANY = [5000, 60, 2047, 61, 90, 2049, 50, 4097, 70, 80]


@pytest.mark.parametrize("sums", ["random", "few"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("keep,sinks,recent", [(40, 4, 8), (2040, 0, 100), (2046, 2000, 46), (4090, 3, 0)])
def test_many_heads(keep, sinks, recent, hd, sums):
    Long(MANY, layers=4, nh=4, hd=hd, sums=sums).check(list(range(10)), keep, sinks, recent)


# Sums that stay in global memory, where places are written while the same row is read: rows wider than 8192 with many blocks,
# wider than 40960 with few.
@pytest.mark.parametrize("keep", [30, 2500, 4999, 4096])
def test_many_heads_of_wide_sums(keep):
    for sums in ("random", "few"):
        Long(MANY, layers=4, nh=4, width=8193, sums=sums).check(list(range(10)), keep, 2, 5)


@pytest.mark.parametrize("keep", [300, 9000, 8192, 16383, 20998])
def test_few_heads_of_very_wide_sums(keep):
    for sums in ("random", "ties"):
        Long([21000, 16384], width=41000, sums=sums).check([1, 0], keep, 3, 11)


def test_a_row_as_wide_as_its_sums():
    Long([40960], sums="few").check([0], 20000, 0, 9)
    Long([40961], sums="few").check([0], 40959, 1, 0)
