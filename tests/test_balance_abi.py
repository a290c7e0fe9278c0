"""The balance-loss entry points check their arguments on the host, before any HIP call (CPU), and the data-parallel counts
(two processes over gloo)."""
import ctypes
import os
import socket
import subprocess
import sys

import pytest

from detr_amd import _lib
from detr_amd._lib import DmRouterSet, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WORD = 0x1000          # an address that is checked and never followed


def sets_of(*queries, experts=None, stride=0):
    arr = (DmRouterSet * max(len(queries), 1))()
    for s, q in enumerate(queries):
        arr[s].logits, arr[s].grad, arr[s].Q, arr[s].image_stride = WORD, WORD, q, stride
        arr[s].experts = experts
    return arr


def loss(sets, S, B=2, E=8, k=2, dtype=0, scores=0, per_image=0, balance=WORD, z=WORD, counts=WORD, slope=WORD, inv=WORD,
         workspace=0x10000, size=1 << 40, status=WORD):
    return lib.dm_balance_loss(sets, S, B, E, k, dtype, scores, per_image, None, balance, z, counts, slope, inv, workspace, size,
                               status, None)


def test_layout():
    assert ctypes.sizeof(DmRouterSet) == 48 and DmRouterSet.image_stride.offset == 32 and DmRouterSet.Q.offset == 40


def test_arguments_are_refused():
    one = sets_of(5)
    bad, big = _lib.E_INVALID_ARG, _lib.E_UNSUPPORTED
    assert loss(one, -1) == bad and loss(None, 1) == bad and loss(one, 1, B=-1) == bad
    assert loss(one, 1, E=0) == bad and loss(one, 1, E=1025) == big
    assert loss(one, 1, k=0) == bad and loss(one, 1, k=9) == bad
    assert loss(one, 1, dtype=3) == bad and loss(one, 1, scores=2) == bad
    assert loss(sets_of(-1), 1) == bad
    assert loss(sets_of(1 << 30), 1) == big                                   # B * Q rows beyond 32 bits
    assert loss(sets_of(5, stride=39), 1) == bad                              # images that overlap
    for what in ("balance", "z", "counts", "slope", "inv", "workspace", "status"):
        assert loss(one, 1, **{what: None}) == bad, what
    assert loss(one, 1, workspace=0x10008) == bad
    need = lib.dm_balance_workspace(one, 1, 2, 8, 0)
    assert need > 0 and loss(one, 1, size=need - 1) == bad
    both = sets_of(5, 5)
    both[1].experts = WORD                                                    # given for one set, not for the other
    assert loss(both, 2) == bad
    # more workgroups than a launch has threads for: images by themselves, and images that are not dense
    assert loss(sets_of(2), 1, B=1 << 22, per_image=1) == big and loss(sets_of(2, stride=99), 1, B=1 << 24) == big
    one[0].logits = None
    assert loss(one, 1) == bad
    assert lib.dm_balance_workspace(one, 1, 2, 0, 0) == bad and lib.dm_balance_workspace(one, 1, 2, 4096, 0) == big


def test_nothing_to_do():
    assert loss(None, 0) == 0
    assert loss(sets_of(5), 1, B=0, per_image=1, balance=None, z=None, counts=None, slope=None, inv=None, workspace=None) == 0
    assert lib.dm_expert_counts(None, 0, 2, 8, 2, 0, 0, None, None, 0, None, None) == 0
    assert lib.dm_balance_backward(None, 0, 2, 8, 0, 0, 0, None, None, None, None, None) == 0


def test_backward_arguments_are_refused():
    one = sets_of(5)
    bad = _lib.E_INVALID_ARG

    def back(sets=one, S=1, E=8, dtype=0, scores=0, slope=WORD, inv=WORD, gz=WORD):
        return lib.dm_balance_backward(sets, S, 2, E, dtype, scores, 0, slope, inv, WORD, gz, None)

    assert back(S=-1) == bad and back(E=0) == bad and back(dtype=-1) == bad and back(scores=5) == bad
    assert back(slope=None) == bad and back(inv=None) == bad
    assert back(scores=1) == bad                                              # sigmoid scores have no z
    assert lib.dm_balance_backward(sets_of(2, stride=99), 1, 1 << 24, 8, 0, 0, 0, WORD, WORD, WORD, WORD, None) == _lib.E_UNSUPPORTED
    one[0].grad = None
    assert back() == bad
    # the counts alone are those of logits
    given = sets_of(5, experts=WORD)
    assert lib.dm_expert_counts(given, 1, 2, 8, 2, 0, 0, WORD, 0x10000, 1 << 40, WORD, None) == bad


def test_cpu_tensors_are_refused():
    import torch

    from detr_amd import losses

    with pytest.raises(RuntimeError, match="GPU"):
        losses.balance_losses(torch.zeros(1, 2, 3), 1)
    with pytest.raises(RuntimeError, match="GPU"):
        losses.expert_counts(torch.zeros(1, 2, 3), 1)


WORKER = """
import sys, torch, torch.distributed as dist
sys.path.insert(0, {root!r})
rank = int(sys.argv[1])
dist.init_process_group("gloo", init_method="tcp://127.0.0.1:{port}", rank=rank, world_size=2)
from detr_amd import dist as ddist
mine = torch.arange(6).view(1, 6) * (rank + 1)
total = ddist.all_reduce_expert_counts(mine)
assert total.tolist() == [[0, 3, 6, 9, 12, 15]], total
assert mine.tolist() == [[(rank + 1) * i for i in range(6)]], mine
dist.destroy_process_group()
"""


def test_counts_of_two_ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    code = WORKER.format(root=ROOT, port=port)
    ranks = [subprocess.Popen([sys.executable, "-c", code, str(r)], stderr=subprocess.PIPE, text=True) for r in range(2)]
    for r in ranks:
        _, err = r.communicate(timeout=120)
        assert r.returncode == 0, err
