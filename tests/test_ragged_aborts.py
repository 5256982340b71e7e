"""What the ragged attention kernels do after a bounded wait has run out, without a
GPU: the warps of a CTA leave together, and no copy is in flight when it exits.

The second part replays the producer warps' accounting on mbarriers (phases and
transaction bytes).  Another warp's wait runs out, or one of the producer's own,
at any point; copies land at any time.  Afterwards every copy that was issued has
landed, and no wait named a phase that its barrier had left behind (the hardware
would take the next phase of the same parity for it and wait in vain)."""
import os
import random
import re

import pytest

from tests.flash_pipeline_model import Bar

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-vl_b200", "csrc")


def test_a_warp_reads_the_abort_flag_with_one_vote():
    """The flag is set by other warps at any time, so lanes that read it for
    themselves may part, and the rest of the warp then waits for them in a shuffle."""
    src = open(os.path.join(CSRC, "ragged_prefill.cu")).read()
    reads = [m.start() for m in re.finditer(r"\*abort_flag(?!\s*=[^=])", src)
             if not src[:m.start()].endswith("volatile int")]
    assert reads
    for at in reads:
        line = src[src.rfind("\n", 0, at) + 1:src.find("\n", at)]
        assert src[:at].endswith("__any_sync(0xffffffffu, "), line.strip()


class Copies:
    """Barriers of a CTA and the bulk copies in flight onto them."""

    def __init__(self, seed):
        self.rng = random.Random(seed)
        self.flying = []          # (bar, bytes)
        self.lapped = 0

    def issue(self, bar, nbytes, parts=4):
        bar.arrive_expect_tx(nbytes)
        self.flying += [(bar, nbytes // parts)] * parts

    def land(self, bar=None):
        """Some copies land, or all onto one barrier."""
        keep = []
        for b, n in self.flying:
            if b is bar or (bar is None and self.rng.random() < 0.3):
                b.complete_tx(n)
            else:
                keep.append((b, n))
        self.flying = keep

    def wait(self, bar, phase):
        """A parity wait that ends as soon as the copies onto its barrier land."""
        self.land(bar)
        if bar.phase != phase + 1:
            self.lapped += 1      # the parity of a later phase, or one never armed

    def patience(self):
        """Whether a wait for another warp returns (else it has run out)."""
        self.land()
        return self.rng.random() > 0.03


def prefill_producer(c: Copies, mended: bool):
    """Warp 0 of ragged_prefill_kernel.  Returns what its last waits left behind."""
    rng = c.rng
    q_full, v_tail = Bar("q_full", 1), Bar("v_tail", 1)
    k_full = [Bar(f"k_full{i}", 1) for i in range(2)]
    v_full = [Bar(f"v_full{i}", 1) for i in range(2)]
    T = ic = nk = nv = tails = 0
    ok = True
    while ok and rng.random() > 0.05:                  # an abort flag or no more items
        if ic >= 1 and not c.patience():               # q_empty
            ok = False
            break
        if ic >= 1:
            c.land(q_full)
        c.issue(q_full, 4096)
        ic += 1
        n, tail = rng.randint(1, 5), rng.random() < 0.6
        for j in range(n):
            s = T & 1
            if T >= 2 and not c.patience():            # k_empty: its MMAs have read the copy
                ok = False
                break
            if T >= 2:
                c.land(k_full[s])
            c.issue(k_full[s], 32768)
            nk = T + 1
            if T >= 2 and not c.patience():            # v_empty
                ok = False
                break
            if T >= 2:
                c.land(v_full[s])
            if tail and j == n - 1:
                c.issue(v_tail, 32768)
                tails += 1
                if rng.random() < 0.03:                # its own wait runs out
                    ok = False
                    break
                c.wait(v_tail, tails - 1)
                v_full[s].arrive()
                if mended:
                    nv = T + 1
            else:
                c.issue(v_full[s], 32768)
                nv = T + 1
            T += 1
    if mended or not ok:
        if ic > 0:
            c.wait(q_full, ic - 1)
        for j in range(max(0, nk - 2), nk):
            c.wait(k_full[j & 1], j >> 1)
        for j in range(max(0, nv - 2), nv):
            c.wait(v_full[j & 1], j >> 1)
        if tails > 0:
            c.wait(v_tail, tails - 1)
    return len(c.flying), c.lapped


def decode_producer(c: Copies, mended: bool, stages=6):
    """The producer warp of ragged_decode_kernel."""
    full = [Bar(f"full{i}", 1) for i in range(stages)]
    it, ok = 0, True
    for _ in range(c.rng.randint(1, 40)):
        if it >= stages and not c.patience():          # empty[s]
            ok = False
            break
        if it >= stages:
            c.land(full[it % stages])
        c.issue(full[it % stages], 32768)
        it += 1
    if mended or not ok:
        for i in range(max(0, it - stages), it):
            c.wait(full[i % stages], i // stages)
    return len(c.flying), c.lapped


@pytest.mark.parametrize("producer", [prefill_producer, decode_producer])
def test_every_copy_has_landed_when_the_cta_exits(producer):
    runs = [producer(Copies(seed), True) for seed in range(3000)]
    assert all(r == (0, 0) for r in runs)
    # waiting only after a wait of its own had run out left copies in flight, and V
    # tiles that end inside a request were not counted
    old = [producer(Copies(seed), False) for seed in range(3000)]
    assert any(flying for flying, _ in old)
    if producer is prefill_producer:
        assert any(lapped for _, lapped in old)
