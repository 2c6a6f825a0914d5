"""What the operators around a head do at their edges, as far as it needs no GPU."""
import random
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests.test_head_ops_cpu import P, SHAPE, _caller

CSRC = Path(__file__).resolve().parent.parent / "addernetcuda_b200" / "csrc"

RING = r"""
#include "ring.h"
#include <cstdio>
#include <cstdlib>

// Barriers of one arrival a phase, whose arrivals come some time after they were asked for, in order; a waiter may let `patience` of them come.
template <int STAGES> int run(int uses, int delivered, int patience, bool& drained, bool& early) {
    int over[STAGES] = {}, begun[STAGES] = {}, came = 0, stage = 0, turn = 0;
    const auto come = [&] { if (came < uses) { ++over[came % STAGES]; ++came; return true; } return false; };
    for (int use = 0; use < uses; ++use) {      // the producer: a stage's use begins when the one before is over
        while (over[stage] < begun[stage]) come();
        ++begun[stage];
        if (++stage == STAGES) { stage = 0; ++turn; }
    }
    while (came < delivered) come();
    drained = adder::ring_drain<STAGES>(stage, turn, [&](int i, unsigned parity) {
        while ((unsigned)(over[i] & 1) == parity)      // the phase of that parity is not over
            if (patience-- <= 0 || !come()) return false;
        return true;
    });
    early = drained && came < uses;
    return came;
}
template <int STAGES> void all() {
    for (int uses = 0; uses <= 4 * STAGES + 1; ++uses)
        for (int delivered = 0; delivered <= uses; ++delivered) {
            bool drained, early;
            const int came = run<STAGES>(uses, delivered, 1 << 20, drained, early);
            if (!drained || early || came != uses) { std::printf("%d stages, %d uses, %d over: left with %d\n", STAGES, uses, delivered, came); std::exit(1); }
            run<STAGES>(uses, uses, 0, drained, early);
            if (!drained) { std::printf("%d stages, %d uses: waits for what never comes\n", STAGES, uses); std::exit(1); }
            for (int patience = 0; patience < STAGES; ++patience) {
                run<STAGES>(uses, delivered, patience, drained, early);
                if (early) { std::printf("%d stages, %d uses, %d over: left early\n", STAGES, uses, delivered); std::exit(1); }
            }
        }
}
int main() { all<1>(); all<2>(); all<5>(); all<6>(); }
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_a_ring_is_left_when_its_last_uses_are_over(tmp_path):
    """The word that a stage is free goes to shared memory, whenever it is ready: a thread that has walked through the ring waits for the last word of
    every stage, for no earlier one (whose parity may be the same) and for none that never comes."""
    (tmp_path / "ring.cpp").write_text(RING)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "ring.cpp"), "-o", str(tmp_path / "ring")], check=True)
    done = subprocess.run([str(tmp_path / "ring")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_temperatures_too_small_for_their_inverse():
    """1 / T beyond fp32: 0 times infinity would be NaN.  The smallest that are taken have an inverse."""
    fwd = _caller("adder_b200_distillation_forward", x=P, t=0, rows=2, v=10, xs=10, z=P, zt=0, at=P, k=3, tau=1.0, tg=None, ig=-100, d=P, lp=None, st=None, ma=None, s=None)
    bwd = _caller("adder_b200_distillation_backward", x=P, t=0, rows=2, v=10, xs=10, at=P, k=3, tau=1.0, tg=None, ig=-100, st=P, ma=P, gd=P, gl=None, dx=P, s=None)
    for tau in (1e-45, 1e-40, 4.2e-39):
        assert fwd(tau=tau) == bwd(tau=tau) == SHAPE
    for tau in (4.3e-39, 1e-37, 3e38):
        assert fwd(tau=tau, rows=0) == bwd(tau=tau, rows=0) == 0


def test_rows_of_views():
    """Rows are found where a view of the same memory has them, and copied otherwise."""
    from addernetcuda_b200.layernorm import _rows
    rng = random.Random(0)
    kept = 0
    for _ in range(3000):
        shape = [rng.choice([1, 2, 3, 5]) for _ in range(rng.randint(1, 4))]
        t = torch.arange(20000).as_strided([s * rng.choice([1, 2]) for s in shape], torch.empty([2 * s for s in shape]).stride(), rng.choice([0, 1, 5]))
        t = t[tuple(slice(rng.choice([0, 1]) if n > 1 else 0, n, rng.choice([1, 1, 2])) for n in t.shape)]
        if rng.random() < 0.4:
            t = t.permute(rng.sample(range(t.dim()), t.dim()))
        if rng.random() < 0.2:
            t = t[:1].expand(3, *t.shape[1:])
        d = 1
        for n in t.shape[t.dim() - rng.randint(1, t.dim()):]:
            d *= n
        rows = t.numel() // d
        v, stride = _rows(t, rows, d)
        got = torch.as_strided(v, (rows, d), (stride, 1), v.storage_offset())
        assert torch.equal(got, t.reshape(rows, d))
        try:
            view = t.view(rows, d)
            same = d == 1 or view.stride(1) == 1
        except RuntimeError:
            same = False
        assert (v.data_ptr() == t.data_ptr()) == same
        kept += same and not t.is_contiguous()
    assert kept > 100


TRACED = """
import torch
from addernetcuda_b200.layernorm import _rows
class Copy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return torch.zeros_like(x, memory_format=torch.contiguous_format) if _rows(x, x.numel() // x.shape[-1], x.shape[-1])[1] else None
class Net(torch.nn.Module):
    def forward(self, x):
        return Copy.apply(x.movedim(-3, -1))
x = torch.randn(2, 3, 4, 5)
assert torch.jit.trace(Net(), x, check_trace=False)(x).shape == (2, 4, 5, 3)
"""


def test_rows_that_are_copied_in_a_trace():
    """In a process of its own, which a trace with a refused view in it ended."""
    done = subprocess.run([sys.executable, "-c", TRACED], capture_output=True, text=True, timeout=300, cwd=CSRC.parent.parent)
    assert done.returncode == 0, done.stderr[-2000:]
