"""The library's scratch of tree attention and log probabilities: given back when
a host thread ends, refused to grow inside a capture, and kept for as long as a
captured call may be replayed."""
import threading
import time

import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda
from test_gpu_logprobs import _check
from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


def _logits_call(torch, x, top, ids, stream=0):
    V.logprobs(x.data_ptr(), x.shape[0], x.shape[1], top_k=top.shape[1], top_logprobs=top.data_ptr(),
               top_ids=ids.data_ptr(), stream=stream)


@pytest.mark.parametrize("call,threads", [("tree_attention", 30), ("logprobs", 150)])
def test_threads_that_end_give_their_scratch_back(call, threads):
    """30 threads with 40 MB each, 150 with 156 KB."""
    torch = torch_cuda()
    if call == "tree_attention":
        case = Case(torch, np.random.default_rng(1), [30], [60], 8, 1, 128, 16, "f16", "f32")
        table = np.zeros((1, (1 << 16) // 16), dtype=np.int32)
        table[:, :case.table.shape[1]] = case.table
        case.table = table
        out = torch.empty_like(case.q)
        need = V.lib.vspec_b200_tree_attention_workspace_bytes(1, 60, 60, 8, 1, 128, 1 << 16)
        run = lambda: case.run(out=out, max_ctx=1 << 16)  # noqa: E731
    else:
        x = torch.randn((64, 151936), device="cuda")
        top, ids = torch.empty((64, 32), device="cuda"), torch.empty((64, 32), dtype=torch.int32, device="cuda")
        need = V.lib.vspec_b200_logprobs_workspace_bytes(64, 151936, 32)
        run = lambda: _logits_call(torch, x, top, ids)  # noqa: E731
    run()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    wrong = []

    def work():
        try:
            torch.cuda.set_device(0)
            run()
            torch.cuda.synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    for _ in range(threads):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert not wrong
    kept = need * threads
    for _ in range(50):          # join() returns a little before a thread's own objects are gone
        kept = before - torch.cuda.mem_get_info()[0]
        if kept < need * threads / 4:
            break
        time.sleep(0.1)
    print(f"{call}: {need} bytes a thread, {kept} kept after {threads} threads")
    assert kept < need * threads / 4


def test_no_growth_inside_a_capture():
    torch = torch_cuda()
    x = torch.randn((3, 60000), device="cuda")
    top, ids = torch.empty((3, 4), device="cuda"), torch.empty((3, 4), dtype=torch.int32, device="cuda")
    y, seen = torch.zeros(8, device="cuda"), []

    def work():
        torch.cuda.set_device(0)
        g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=st):
            try:
                _logits_call(torch, x, top, ids, stream=st.cuda_stream)
            except V.VspecB200Error as e:
                seen.append(str(e))
            y.add_(1.0)
        g.replay()
        torch.cuda.synchronize()

    t = threading.Thread(target=work)    # a thread without scratch
    t.start()
    t.join()
    assert len(seen) == 1 and "d_workspace" in seen[0]
    assert (y == 1.0).all()              # the capture went on


def test_scratch_of_a_captured_call_outlives_larger_calls_and_its_thread():
    torch = torch_cuda()
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((3, 60000), device="cuda", generator=gen)
    top, ids = torch.empty((3, 4), device="cuda"), torch.empty((3, 4), dtype=torch.int32, device="cuda")
    case = Case(torch, np.random.default_rng(2), [3000], [4], 4, 1, 128, 16, "f16", "f32")
    expect = case.run().clone()
    out, big = torch.empty_like(expect), []
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()

    def work():
        torch.cuda.set_device(0)
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            _logits_call(torch, x, top, ids, stream=st.cuda_stream)
            case.run(out=out, stream=st.cuda_stream)
            st.synchronize()
            table, ctx, cu, mask = case._keep
            with torch.cuda.graph(g, stream=st):
                _logits_call(torch, x, top, ids, stream=st.cuda_stream)
                V.tree_attention(case.q.data_ptr(), case.codes[0].data_ptr(), case.codes[1].data_ptr(), None, None,
                                 table.data_ptr(), ctx.data_ptr(), cu.data_ptr(), mask.data_ptr(), out.data_ptr(), 1, 4, 4,
                                 4, 1, 128, 16, case.table.shape[1], case.pages, case.max_ctx, case.scale,
                                 mask_words=case.words, stream=st.cuda_stream)
            st.synchronize()
            # calls whose scratch is larger, and allocations that would take a freed one's place
            more = torch.randn((64, 151936), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
            a, b = torch.empty((64, 32), device="cuda"), torch.empty((64, 32), dtype=torch.int32, device="cuda")
            _logits_call(torch, more, a, b, stream=st.cuda_stream)
            wide = Case(torch, np.random.default_rng(3), [30, 3000], [60, 60], 8, 1, 128, 16, "f16", "f32")
            wide.run(stream=st.cuda_stream)
            st.synchronize()
            big.extend([more, a, b, wide])

    t = threading.Thread(target=work)
    t.start()
    t.join()
    time.sleep(0.5)
    big.extend(torch.full((1 << 22,), -1, dtype=torch.int32, device="cuda") for _ in range(8))
    for _ in range(3):
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect)
        _check(dict(top=top.cpu().numpy(), ids=ids.cpu().numpy()), x.double().cpu().numpy(), None, 4, None, 1.0, entropy=False)
