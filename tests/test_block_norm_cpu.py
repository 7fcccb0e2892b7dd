"""What the block norm calls refuse, before any device work (no GPU needed)."""
import pytest

import blackhole_b200 as bh
from blackhole_b200 import fused

A = 1 << 40          # an aligned address that is never dereferenced: every case is refused first
STEP = 1 << 34


def forward(**over):
    names = ("x", "o", "gate", "weight", "bias", "post_weight", "post_bias", "h", "out", "sf", "stats")
    p = {n: A + i * STEP for i, n in enumerate(names)}
    v = dict(rows=4, H=256, kind="rms", post_norm=True, gate_rows=0, out_format="mxfp8", eps=1e-6,
             scale=1.0, global_scale=1.0, **p)
    v.update(over)
    rows, H, x = v.pop("rows"), v.pop("H"), v.pop("x")
    bh.block_norm(rows, H, x, stream=0, **v)


@pytest.mark.parametrize("over", [
    dict(rows=0), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(H=0), dict(H=12), dict(H=16392), dict(H=264), dict(gate_rows=-1),
    dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(x=None), dict(out=None, h=None, sf=None, weight=None, bias=None),
    dict(o=None), dict(post_norm=False), dict(out=None), dict(sf=None), dict(out_format="bf16"),
    dict(out_format="nvfp4", global_scale=0.0), dict(out_format="nvfp4", global_scale=float("nan")),
    dict(out_format="nvfp4", H=264), dict(x=A + 8), dict(out=A + 8 * STEP + 4), dict(weight=A + 3 * STEP + 2),
    dict(h=A + 16), dict(h=A + STEP), dict(out=A), dict(out=A + STEP + 16), dict(out=A + 7 * STEP),
])
def test_forward_refusals(over):
    with pytest.raises(bh.BlackholeError) as e:
        forward(**over)
    assert e.value.code == 1


def backward(**over):
    names = ("h", "stats", "dx", "dy", "dh", "weight", "o", "do", "post_weight", "post_bias", "gate", "dweight",
             "dbias", "dpost_weight", "dpost_bias", "dgate", "workspace")
    v = {n: A + i * STEP for i, n in enumerate(names)}
    v.update(rows=4, H=256, post_norm=True, gate_rows=0, scale=1.0, workspace_bytes=1 << 30)
    v.update(over)
    rows, H, h, st, dx = (v.pop(k) for k in ("rows", "H", "h", "stats", "dx"))
    bh.block_norm_backward(rows, H, h, st, dx, stream=0, **v)


@pytest.mark.parametrize("over", [
    dict(rows=0), dict(rows=(1 << 30) + 1), dict(H=12), dict(H=16392), dict(gate_rows=-1), dict(scale=float("nan")), dict(h=None),
    dict(stats=None), dict(dx=None), dict(dy=None, dh=None), dict(o=None), dict(do=None),
    dict(post_norm=False), dict(gate=None), dict(workspace_bytes=8), dict(dx=A), dict(dx=A + 3 * STEP),
    dict(dx=A + 4 * STEP + 16), dict(dx=A + 6 * STEP), dict(do=A + 6 * STEP), dict(do=A + 2 * STEP),
    dict(dy=A + 3 * STEP + 8), dict(workspace=A + 16 * STEP + 4),
])
def test_backward_refusals(over):
    with pytest.raises(bh.BlackholeError) as e:
        backward(**over)
    assert e.value.code == 1


def test_names_and_null_arguments():
    with pytest.raises(KeyError):
        forward(kind="batch")
    with pytest.raises(KeyError):
        forward(out_format="fp8")
    L = bh.load()
    assert L.blackhole_sm100_block_norm(None, None) == 1
    assert L.blackhole_sm100_block_norm_backward(None, None) == 1
    ptrs = [A] + [0] * 7 + [A + STEP, 0, 0]
    pack = lambda kind, fmt: fused._NORM.pack(4, 256, kind, 1, 0, 1, 0, 0, fmt, 1e-6, 1.0, 1.0, *ptrs)  # noqa: E731
    for kind, fmt in ((2, 0), (-1, 0), (0, 5), (0, -1)):
        assert L.blackhole_sm100_block_norm(pack(kind, fmt), None) == 1


def test_tensors_are_checked():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        forward(x=torch.zeros(4, 256, dtype=torch.bfloat16))               # not on a GPU
    with pytest.raises(TypeError):
        forward(x="x")


@pytest.mark.parametrize("rows,H,gate,gr", [(1, 8, True, 0), (16384, 8192, True, 0), (16384, 8192, False, 0),
                                            (300, 16384, True, 7), (5, 1000, True, 1)])
def test_workspace_size(rows, H, gate, gr):
    n = bh.block_norm_backward_workspace_bytes(rows, H, gate, gr)
    per = (6 if gate and gr != 1 else 4) * H * 4
    assert n % per == 0 and 1 <= n // per <= min(rows, 148 * 16)
    for bad in ((0, H, gr), ((1 << 30) + 1, H, gr), (rows, H + 4, gr), (rows, 16392, gr), (rows, H, -1)):
        assert bh.block_norm_backward_workspace_bytes(bad[0], bad[1], gate, bad[2]) < 0


def test_structs_match_the_header(tmp_path):
    """The packed arguments have the C structs' sizes and offsets."""
    import os
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "blackhole_sm100.h"\n'
                   "int main(void) {\n"
                   'printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(blackhole_sm100_epilogue),\n'
                   " sizeof(blackhole_sm100_block_norm_args), sizeof(blackhole_sm100_block_norm_backward_args),\n"
                   " offsetof(blackhole_sm100_epilogue, bias), offsetof(blackhole_sm100_block_norm_args, x),\n"
                   " offsetof(blackhole_sm100_block_norm_backward_args, workspace_bytes));\n}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), "-I", os.path.join(cuda, "include"), str(src),
                    "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [fused._EPILOGUE.size, fused._NORM.size, fused._NORM_BACKWARD.size, 16, 48,
                   fused._NORM_BACKWARD.size - 8]
