"""What the binding of the losses over logit rows refuses by itself, because only the tensors can tell: types,
shapes and strides of what is read, room and type of what is written, memory the device does not reach. CPU
only: nothing is launched."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def refused(call, text):
    from geistlib_amd.binding import GeistHipError
    with pytest.raises(GeistHipError) as err:
        call()
    assert err.value.code == 2 and text in str(err.value), str(err.value)


@pytest.mark.parametrize("what", ["loss", "logprob", "entropy", "ratios"])
def test_outputs(what):
    from geistlib_amd import HipSampler
    refused(lambda: HipSampler._output(torch.zeros(7), 8, what), what + ": (7,)")
    refused(lambda: HipSampler._output(torch.zeros(8, dtype=torch.float16), 8, what), "float16")
    refused(lambda: HipSampler._output(torch.zeros(8, dtype=torch.float64), 8, what), "float64")
    refused(lambda: HipSampler._output(torch.zeros(16)[::2], 8, what), "consecutive")
    refused(lambda: HipSampler._output(torch.zeros(8), 8, what), "not in device memory")
    assert HipSampler._output(None, 8, what) is None


def test_workspaces():
    from geistlib_amd import HipSampler
    refused(lambda: HipSampler._scratch(torch.zeros(64, dtype=torch.uint8)[::2]), "not contiguous")
    refused(lambda: HipSampler._scratch(torch.zeros(64, dtype=torch.uint8)), "not in device memory")
    assert HipSampler._scratch(None) == (None, 0)


def test_rows():
    from geistlib_amd import HipSampler
    rows = HipSampler.loss_rows
    x = torch.zeros(4, 10)
    refused(lambda: rows(torch.zeros(4, 1, 1)), "2-D")
    refused(lambda: rows(torch.zeros(4)), "2-D")
    refused(lambda: rows(x.t()), "consecutive")
    refused(lambda: rows(x.double()), "float64")
    refused(lambda: rows(x, grad=torch.zeros(4, 9)), "gradient of (4, 9)")
    refused(lambda: rows(x, grad=torch.zeros(3, 10)), "gradient of (3, 10)")
    refused(lambda: rows(x, grad=torch.zeros(4, 10, dtype=torch.bfloat16)), "bfloat16")
    refused(lambda: rows(x, grad=torch.zeros(10, 4).t()), "consecutive")
    refused(lambda: rows(x, allowed=torch.zeros(2, 1, dtype=torch.int32)), "allowed")
    refused(lambda: rows(torch.zeros(4, 33), allowed=torch.zeros(4, 1, dtype=torch.int32)), "allowed")
    refused(lambda: rows(x, allowed=torch.zeros(4, 1, dtype=torch.int64)), "allowed")
    refused(lambda: rows(x), "logits: not in device memory")
    refused(lambda: rows(torch.zeros(4, 1)), "logits: not in device memory")


def test_descriptions():
    from geistlib_amd import HipSampler
    i, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    ids, values = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, 3)
    refused(lambda: HipSampler.teacher(ids, torch.zeros(4, 2)), "values of (4, 2)")
    refused(lambda: HipSampler.teacher(ids.long(), values), "int64")
    refused(lambda: HipSampler.teacher(ids, torch.zeros(3, 4).t()), "consecutive")
    refused(lambda: HipSampler.teacher(ids, torch.zeros(4, 5)[:, :3]), "one stride")
    refused(lambda: HipSampler.teacher(ids, values), "ids: not in device memory")
    refused(lambda: HipSampler.policy(i.long(), f), "tokens: (4,) torch.int64")
    refused(lambda: HipSampler._vector(torch.zeros(3), 4, "torch.float32", "advantage"), "advantage: (3,)")
    refused(lambda: HipSampler._vector(torch.zeros(8)[::2], 4, "torch.float32", "old"), "consecutive")
    refused(lambda: HipSampler.policy(i, f), "tokens: not in device memory")
    refused(lambda: HipSampler.preference(i, i[:0]), "seq_start: 0 entries")
    refused(lambda: HipSampler.preference(i, i[:1]), "seq_start: 1 entries")
    refused(lambda: HipSampler.preference(i.float(), i[:3]), "tokens")


def test_refusals_do_not_depend_on_assertions():
    code = ("import torch\nfrom geistlib_amd import HipSampler\nfrom geistlib_amd.binding import GeistHipError\n"
            "try:\n    HipSampler._output(torch.zeros(7), 8, 'loss')\nexcept GeistHipError:\n    print('refused')\n")
    p = subprocess.run([sys.executable, "-O", "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert p.stdout.strip() == "refused", p.stdout + p.stderr
