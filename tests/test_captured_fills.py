"""What a captured train step may hold: no memset nodes (replays behind the first have been seen to get them wrong), fills are kernels."""
import glob
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_launch_records_a_memset():
    found = [f for f in glob.glob(os.path.join(ROOT, "wide_deep_amd", "csrc", "*.h*")) if "hipMemset" in open(f).read()]
    assert not found, found


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 1000, 70001])
def test_touched_rows_are_cleared_in_every_replay(rows):
    """wd_adam_untouched clears its bitmap, all of it and nothing behind it, eager and replayed; rows whose bit is set do not move."""
    from wide_deep_amd import capi, hipgraph, plan as plan_
    from wide_deep_amd.engine import WideDeepEngine
    from wide_deep_amd import synth
    spec = plan_.criteo_spec(n_dense=2, n_sparse=1, buckets=rows, dim=16, hidden=(16,))
    spec.dnn_opt, spec.lin_opt = ("Adam", 0.01, 0.9, 0.999, 1e-8), ("Adam", 0.02, 0.9, 0.999, 1e-8)
    eng = WideDeepEngine(spec, max_batch=64, seed=1)
    eng.train_step(synth.to_device_ids(eng.plan, synth.make_raw_batch(eng.plan, 64, seed=1, pos_rate=0.4)))
    torch.cuda.synchronize()
    assert not bool(eng.touched.any())
    words = (rows + 31) // 32
    bits = torch.full((words + 3,), -1, dtype=torch.int32, device="cuda")
    import ctypes
    from wide_deep_amd.capi import call, ptr
    od, ol = ctypes.byref(eng.opt_c["dnn"]), ctypes.byref(eng.opt_c["linear"])

    def launch():
        st = torch.cuda.current_stream().cuda_stream
        call("wd_adam_untouched", ptr(eng.emb), ptr(eng.emb_a), ptr(eng.emb_acc), ptr(eng.wide), ptr(eng.slots_dev), 1, rows, rows, ptr(bits), od, ol, st)

    def check(run):
        bits.fill_(-1)
        emb, wide = eng.emb.clone(), eng.wide.clone()
        run()
        torch.cuda.synchronize()
        assert bits[:words].tolist() == [0] * words and bits[words:].tolist() == [-1] * 3
        assert torch.equal(eng.emb, emb) and torch.equal(eng.wide, wide)

    check(launch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = hipgraph.new_graph()
    with torch.cuda.graph(g, stream=side):
        launch()
    for _ in range(3):
        check(g.replay)
        check(launch)
