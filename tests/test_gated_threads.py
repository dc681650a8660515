"""The record of living eager graphs, used from several threads: no GPU is touched."""
from __future__ import annotations

import sys
import threading

import torch

from helion_b200 import gated


class Node:
    """Stands for a backward node of an eager forward pass."""

    next_functions = ()


def test_a_capture_is_checked_while_other_threads_run_forward_passes():
    leaf = torch.zeros(1, requires_grad=True)
    kept = [Node() for _ in range(1000)]
    for n in kept:
        gated._eager_nodes.add(n)
    stop, failed = threading.Event(), []

    def forward_passes():
        while not stop.is_set():
            short = [Node() for _ in range(50)]
            for n in short:
                gated._eager_nodes.add(n)

    threads = [threading.Thread(target=forward_passes) for _ in range(2)]
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        for t in threads:
            t.start()
        for _ in range(40):
            gated._refuse_capture(leaf)  # refuses nothing: no graph holds the leaf
    except RuntimeError as e:
        failed.append(e)
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
    assert not failed, failed
    del kept, n
    assert not gated._eager_nodes  # the record keeps no graph alive
