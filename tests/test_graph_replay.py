"""Calls that only launch (tgpu_plan_execute, tgpu_plan_traffic, tgpu_conv_execute) in a captured graph: no memset node of the runtime in
them, and every replay equals the eager call -- with the counters of the clean-block pre-pass and the traffic stage's lengths, which
each pass clears for itself, and with other input and eager work between the replays."""
import os
import re

import numpy as np
import pytest

import oraclelib as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "osmo-tetra_amd", "csrc")


def _body(path, head):
    """the text of the C function whose definition starts with head"""
    text = open(os.path.join(CSRC, path)).read()
    i = text.index(head)
    return text[i:text.index("\n}\n", i)]


@pytest.mark.parametrize("path,head", [("tg_host.c", "static int plan_run("), ("tg_host.c", "static int plan_traffic("),
                                       ("tg_traffic.hip", 'extern "C" int tgk_traffic('), ("tg_k_trellis.hip", 'extern "C" int tgk_clean('),
                                       ("tg_k_trellis.hip", 'extern "C" int tgk_conv('), ("tg_conv.c", "int tgpu_conv_execute(")])
def test_launch_only_calls_record_no_memset(path, head):
    assert not re.findall(r"hipMemset\w*\(", _body(path, head))


def _slots(T, n, ber, seed):
    ty = np.random.default_rng(5).choice([O.TRAIN_NORM_1, O.TRAIN_NORM_2, O.TRAIN_SYNC], n, p=[0.45, 0.45, 0.1]).astype(np.uint8)
    ty[0] = O.TRAIN_SYNC
    return ty, T.synth_slots(ty, seed=seed, scramb_init=O.scramb_get_init(262, 42, 1), ber=ber)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 6001])                 # above 4096 slots the two trellis launches fork to a side stream
@pytest.mark.parametrize("fast,traffic", [(True, False), (False, True), (True, True)])
def test_replays_equal_the_eager_call(n, fast, traffic):
    import torch
    import osmo_tetra_amd as T
    eng = T.Engine(0)
    code = np.array([O.scramb_get_init(262, 42, 1)], np.uint32)
    types, quiet = _slots(T, n, 0.0, 11)
    inputs = [quiet, _slots(T, n, 0.03, 12)[1], _slots(T, n, 0.004, 13)[1]]
    offs = np.arange(n, dtype=np.uint64) * T.SLOT_BYTES
    marks = torch.from_numpy(np.random.default_rng(6).choice([0, 1, 3], n).astype(np.uint8)).cuda()
    d_stream = torch.empty(n * T.SLOT_BYTES, dtype=torch.uint8, device="cuda")

    def outputs():
        return (torch.empty(n * T.REC_BYTES, dtype=torch.uint8, device="cuda"), torch.empty(n * 432, dtype=torch.uint8, device="cuda"),
                torch.empty(n * 690, dtype=torch.int16, device="cuda"), torch.empty(n, dtype=torch.int16, device="cuda"))

    def mark(bufs):
        for b, v in zip(bufs, (0, 0xEE, 0x7777, 0x5555)):
            b.fill_(v)

    def make(bufs):
        plan = T.Plan(eng, n, 1)
        plan.set_fastpath(fast)
        plan.load(offs, types, None, code)
        if traffic:
            plan.set_traffic(marks.data_ptr(), bufs[1].data_ptr(), bufs[2].data_ptr(), bufs[3].data_ptr())
        return plan

    def load(k):
        d_stream.copy_(torch.from_numpy(inputs[k].reshape(-1)))

    hs = torch.cuda.current_stream().cuda_stream
    eager, own = outputs(), outputs()
    plan_e, plan_g = make(eager), make(own)
    want = []
    for k in range(len(inputs)):
        load(k)
        mark(eager)
        plan_e.execute(d_stream.data_ptr(), eager[0].data_ptr(), hs)
        torch.cuda.synchronize()
        want.append([b.clone() for b in eager])
    assert not bool((want[0][0] == want[1][0]).all())
    if traffic:
        assert bool((want[1][3] == 0).any()) and bool((want[1][3] == 432).any())
    torch.cuda.synchronize()
    plan_g.execute(d_stream.data_ptr(), own[0].data_ptr(), hs)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        plan_g.execute(d_stream.data_ptr(), own[0].data_ptr(), torch.cuda.current_stream().cuda_stream)
    for k in (1, 1, 0, 2, 1, 0):
        load(k)
        mark(own)
        g.replay()
        torch.cuda.synchronize()
        for got, w in zip(own, want[k]):
            assert bool((got == w).all()), k
        mark(own)                                          # eager work of the same plan and of another between the replays
        plan_g.execute(d_stream.data_ptr(), own[0].data_ptr(), hs)
        plan_e.execute(d_stream.data_ptr(), eager[0].data_ptr(), hs)
        torch.cuda.synchronize()
        assert all(bool((got == w).all()) for got, w in zip(own, want[k]))
    del g
    plan_e.close()
    plan_g.close()
    eng.close()
