"""The two scale re-tiling warps of the GEMM kernels on the CPU model: they alternate groups, and scale slabs may land in any order.  An even
number of raw slots gives every slot to one warp.  With an odd number its rounds alternate between the warps, and a warp that is two
groups ahead waits for a parity that an older round has already completed: it reads a slab that has not landed.  Groups of four K-blocks,
and of two as on the 4-bit path."""
import os
import re

import pytest

from tests.pipeline_model import MMA, PRODUCER, SCALE, Pipeline, Timeout

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipkittensp_b200", "csrc")


class TwoScaleWarps(Pipeline):
    def __init__(self, *args, kpg=4, **kw):
        super().__init__(*args, **kw)
        self.kpg, self.in_flight, self.running = kpg, [], 0

    def producer(self):
        n_stage = n_raw = 0
        for tile in range(self.tiles):
            for kb in range(self.kblocks):
                if kb % self.kpg == 0:
                    r = n_raw % self.R
                    yield from self._wait(self.raw_empty[r], ((n_raw // self.R) & 1) ^ 1, PRODUCER)
                    self.in_flight.append((r, (tile, kb // self.kpg)))
                    n_raw += 1
                s = n_stage % self.S
                yield from self._wait(self.empty[s], ((n_stage // self.S) & 1) ^ 1, PRODUCER)
                self.stage_tag[s] = (tile, kb)
                yield
                self._arrive(self.full[s])
                n_stage += 1

    def memory(self):
        """Slabs land in any order."""
        left = self.tiles * -(-self.kblocks // self.kpg)
        while left:
            if self.in_flight and self.rng.random() < 0.1:
                r, tag = self.in_flight.pop(self.rng.randrange(len(self.in_flight)))
                self.raw_tag[r] = tag
                self._arrive(self.raw_full[r])
                left -= 1
            if self.abort:
                return
            yield

    def scale_warp(self, warp):
        n_grp = 0
        for tile in range(self.tiles):
            for grp in range(-(-self.kblocks // self.kpg)):
                if n_grp % 2 == warp:
                    r, g = n_grp % self.R, n_grp % self.G
                    yield from self._wait(self.raw_full[r], (n_grp // self.R) & 1, SCALE)
                    assert self.raw_tag[r] == (tile, grp), "scale warp read a slab of another group"
                    self.raw_tag[r] = None
                    self._arrive(self.raw_empty[r])
                    yield from self._wait(self.atom_empty[g], ((n_grp // self.G) & 1) ^ 1, SCALE)
                    assert self.atom_tag[g] is None, "scale atoms overwritten before the MMA used them"
                    self.atom_tag[g] = (tile, grp)
                    self._arrive(self.atom_full[g])
                n_grp += 1

    def mma(self):
        n_kb = n_grp = 0
        for tile in range(self.tiles):
            for kb in range(self.kblocks):
                s, g = n_kb % self.S, n_grp % self.G
                if kb % self.kpg == 0:
                    yield from self._wait(self.atom_full[g], (n_grp // self.G) & 1, MMA)
                    assert self.atom_tag[g] == (tile, kb // self.kpg), "MMA used the scale atoms of another group"
                yield from self._wait(self.full[s], (n_kb // self.S) & 1, MMA)
                assert self.stage_tag[s] == (tile, kb)
                yield
                self._arrive(self.empty[s])
                if kb % self.kpg == self.kpg - 1 or kb == self.kblocks - 1:
                    self.atom_tag[g] = None
                    self._arrive(self.atom_empty[g])
                    n_grp += 1
                n_kb += 1

    def run(self):
        roles = {"producer": self.producer(), "memory": self.memory(), "scale0": self.scale_warp(0), "scale1": self.scale_warp(1), "mma": self.mma()}
        timed_out = {}
        while roles:
            name = self.rng.choice(sorted(roles))
            try:
                next(roles[name])
            except StopIteration:
                del roles[name]
            except Timeout as t:
                timed_out[name] = t.role
                del roles[name]
        return timed_out


@pytest.mark.parametrize("kpg", [4, 2])
@pytest.mark.parametrize("kblocks,stages,slots,groups", [(64, 4, 2, 3), (64, 5, 2, 3), (33, 4, 2, 3), (64, 11, 4, 4), (7, 8, 4, 4), (64, 16, 8, 4)])
def test_even_numbers_of_slots_hold(kblocks, stages, slots, groups, kpg):
    for seed in range(6):
        assert TwoScaleWarps(2, kblocks, stages=stages, raw_slots=slots, atom_groups=groups, seed=seed, kpg=kpg).run() == {}


def test_an_odd_number_of_slots_does_not():
    def fails(seed):
        try:
            return bool(TwoScaleWarps(2, 64, stages=16, raw_slots=3, atom_groups=4, seed=seed, wait_budget=2000).run())
        except AssertionError:
            return True
    assert any(fails(seed) for seed in range(20))


def test_the_kernels_refuse_to_compile_with_an_odd_number():
    for name in ("gemm_kernel.cuh", "gemm_kernel_2cta.cuh"):
        src = open(os.path.join(CSRC, name)).read()
        assert re.search(r"static_assert\(RAW_SLOTS % 2 == 0", src), name
