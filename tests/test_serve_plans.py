"""The launch plans of the paged attention's test shapes, on the CPU: every shape of
serve_shapes.py gets the kernel that it stands for, and every kernel has a shape."""
import os
import subprocess

import pytest

import serve_shapes as sh

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")


@pytest.fixture(scope="module")
def plan():
    r = subprocess.run(["make", "-s", "-C", NATIVE, "paged"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]

    def show(kind, *args):
        out = subprocess.run([os.path.join(NATIVE, "cbq_paged_host"), kind, *map(str, args)],
                             capture_output=True, text=True, timeout=60, check=True).stdout.split()
        return dict(zip(out[::2], map(int, out[1::2])))
    return show


def test_prompts(plan):
    kernels = set()
    for *shape, rt, streams, parts in sh.PROMPTS:
        p = plan("prompt", *sh.prompt_plan_args(*shape))
        assert (p["rt"], p["streams"], p["parts"] > 1) == (rt, streams, parts), (shape, p)
        kernels.add((shape[0], shape[1], rt, streams))
    # rows of 1 KiB have one stream, rows of up to 256 bytes 128 rows a block
    want = {(hd, size, rt, streams) for hd in (64, 128, 256) for size in (2, 4) for rt in (0, 1, 2)
            for streams in (1, 2) if (rt > 0 or streams == 1) and (rt < 2 or hd * size <= 256)
            and (streams == 1 or hd * size <= 512)}
    assert kernels == want


@pytest.mark.parametrize("i,hd", list(enumerate((64, 128, 256))))
def test_decodes(plan, i, hd):
    for *shape, rt, prefix_parts, own_parts in sh.DECODES:
        p = plan("decode", *sh.decode_plan_args(hd, *shape))
        assert not p["joint"] and p["rt"] == rt[i], (shape, p)
        assert prefix_parts is None or (p["pre_parts"] > 1) == prefix_parts, (shape, p)
        assert (p["own_parts"] > 1) == own_parts, (shape, p)


@pytest.mark.parametrize("hd", (64, 128, 256))
def test_merges(plan, hd):
    for shape in sh.MERGES:
        p = plan("decode", *sh.decode_plan_args(hd, *shape))
        assert p["pre_parts"] + p["own_parts"] > 16 and len(shape[1]) * 2 * shape[3] >= 4096, (shape, p)


@pytest.mark.parametrize("i,hd", list(enumerate((64, 128, 256))))
def test_joints(plan, i, hd):
    """Large batches of few keys behind a prefix read it once for all of them."""
    for *shape, joint in sh.JOINTS:
        p = plan("decode", *sh.decode_plan_args(hd, *shape))
        assert p["joint"] == joint[i], (shape, p)
