"""What the step's calls refuse, before any CUDA call: the C ABI on addresses that are never followed, the Python mirror on CPU tensors."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from gevva_b200 import attention as attn
from gevva_b200 import step
from tests import test_attention_refusals as refusals

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, TOO_LARGE = -3, -6
AT = [n << 30 for n in range(1, 20)]  # apart


@pytest.fixture(scope="module")
def lib():
    if torch.cuda.is_available():
        pytest.skip("calls that are not refused would be launched")
    return step._lib()


def plan(lib, lengths=AT[0], news=AT[1], shift=AT[2], table=AT[3], pool=AT[4], taken=AT[5], offsets=AT[6], after=AT[7], slots=AT[8], positions=AT[9],
         taken_out=AT[10], sequences=5, width=4, stride=6, pages=100, page=16, tokens=40):
    return lib.gevva_step_plan(step._PLAN.pack(lengths or 0, news or 0, shift or 0, table or 0, pool or 0, taken or 0, offsets or 0, after or 0, slots or 0,
                                               positions or 0, taken_out or 0, 0, sequences, width, stride, pages, page, tokens), None)


def trim(lib, lengths=AT[0], keep=AT[1], table=AT[3], pool=AT[4], taken=AT[5], after=AT[7], taken_out=AT[10], sequences=5, width=4, stride=6, pages=100,
         page=16, reserved=0):
    return lib.gevva_step_trim(step._TRIM.pack(lengths or 0, keep or 0, table or 0, pool or 0, taken or 0, after or 0, taken_out or 0, 0, sequences, width,
                                               stride, pages, page, reserved), None)


def append(lib, q=(AT[0], 512, 64), k=(AT[1], 512, 64), v=(AT[2], 512, 64), cache=None, slots=AT[3], positions=AT[4], stride=100, frequencies=AT[5], qw=AT[6],
           kw=AT[7], q_out=AT[8], k_out=None, v_out=None, tokens=3, heads=4, kv_heads=2, dim=64, rotated=64, axes=2, eps=1e-6):
    return lib.gevva_step_append(step._APPEND_AT.pack(*q, *k, *v, ctypes.addressof(cache or refusals.CACHE), slots or 0, positions or 0, stride,
                                                      frequencies or 0, qw or 0, kw or 0, q_out or 0, k_out or 0, v_out or 0, 0, tokens, heads, kv_heads, dim,
                                                      rotated, axes, 0, eps), None)


def sample(lib, logits=AT[0], stride=100, uniforms=AT[1], temperature=AT[2], top_k=AT[3], top_p=AT[4], min_p=AT[5], tokens=AT[6], shares=AT[7], rows=3,
           vocabulary=100, f32=1, softcap=0.0):
    return lib.gevva_step_sample(step._SAMPLE.pack(logits or 0, stride, uniforms or 0, temperature or 0, top_k or 0, top_p or 0, min_p or 0, tokens or 0,
                                                   shares or 0, rows, vocabulary, f32, softcap), None)


def test_what_is_not_refused(lib):
    """(Without a device these end with a CUDA error instead.)"""
    for ok in (plan(lib), plan(lib, after=AT[0], taken_out=AT[5]), plan(lib, shift=None), plan(lib, tokens=0, slots=None, positions=None), trim(lib),
               trim(lib, after=AT[0], taken_out=AT[5]), append(lib), append(lib, axes=1, stride=-5), append(lib, stride=0), append(lib, rotated=0, frequencies=None),
               append(lib, q=(AT[0], 256, 64), q_out=AT[0]), sample(lib), sample(lib, stride=0), sample(lib, temperature=None, top_k=None, top_p=None, min_p=None,
                                                                                                       shares=None), sample(lib, f32=0, logits=AT[0] + 2)):
        assert ok not in (BAD, TOO_LARGE)
    assert sample(lib, rows=0, logits=None) == 0 and append(lib, tokens=0) == 0


SEQUENCES = [dict(lengths=None), dict(lengths=AT[0] + 2), dict(table=None), dict(pool=None), dict(pool=AT[4] + 1), dict(taken=None), dict(after=None),
             dict(taken_out=None), dict(sequences=0), dict(sequences=-1), dict(width=0), dict(stride=3), dict(pages=0), dict(page=8), dict(page=48), dict(page=0),
             dict(width=1 << 27, stride=1 << 27), dict(after=AT[0] + 4), dict(taken_out=AT[0]), dict(after=AT[3] + 4 * 27), dict(taken_out=AT[7] + 16)]


@pytest.mark.parametrize("change", SEQUENCES + [dict(news=None), dict(shift=AT[2] + 2), dict(offsets=None), dict(offsets=AT[6] + 3), dict(tokens=-1),
                                                dict(tokens=(1 << 30) + 1), dict(slots=None), dict(positions=None), dict(after=AT[1]), dict(offsets=AT[0] + 16),
                                                dict(slots=AT[4] + 396), dict(positions=AT[8] + 156), dict(table=AT[4] + 4), dict(slots=AT[5] - 156),
                                                dict(positions=AT[2])])
def test_plan(lib, change):
    assert plan(lib, **change) == BAD


@pytest.mark.parametrize("change", SEQUENCES + [dict(keep=None), dict(keep=AT[1] + 1), dict(reserved=1), dict(after=AT[1]), dict(pool=AT[3] + 4), dict(pool=AT[0] + 16)])
def test_trim(lib, change):
    assert trim(lib, **change) == BAD


def test_more_requests_than_a_plan_has(lib):
    assert plan(lib, sequences=step.MAX_REQUESTS + 1) == TOO_LARGE and trim(lib, sequences=step.MAX_REQUESTS + 1) == TOO_LARGE


@pytest.mark.parametrize("change", refusals.SHAPES[:8] + [dict(q=(AT[0] + 8, 512, 64)), dict(q=(AT[0], 516, 64)), dict(k=(AT[1] + 2, 512, 64)),
                                                         dict(cache=refusals.cache(keys=None)), dict(cache=refusals.cache(page_size=48)),
                                                         dict(cache=refusals.cache(key_slot_stride=100)), dict(slots=None), dict(slots=AT[3] + 2),
                                                         dict(positions=None), dict(positions=AT[4] + 1), dict(axes=0), dict(axes=17), dict(stride=-1),
                                                         dict(stride=1 << 38), dict(frequencies=None), dict(frequencies=AT[5] + 4), dict(rotated=80),
                                                         dict(rotated=8), dict(eps=-1.0), dict(q_out=None), dict(k_out=AT[9]), dict(qw=AT[6] + 2),
                                                         # outputs over what is read
                                                         dict(q_out=AT[0]), dict(q_out=AT[3] - 16), dict(q_out=AT[4] + 400), dict(q_out=AT[5] + 496),
                                                         dict(q_out=AT[6] + 112), dict(q_out=AT[7] - 1520), dict(k_out=AT[1] + 16, v_out=AT[9]),
                                                         dict(k_out=AT[9], v_out=AT[4])])
def test_append(lib, change):
    assert append(lib, **change) == BAD


def test_a_cache_of_more_slots_than_a_whole_number_holds(lib):
    big = refusals.cache(pages=1 << 28, page_size=16)
    assert append(lib, cache=big) == TOO_LARGE


@pytest.mark.parametrize("change", [dict(logits=None), dict(logits=AT[0] + 2), dict(logits=AT[0] + 1, f32=0), dict(uniforms=None), dict(uniforms=AT[1] + 2),
                                    dict(temperature=AT[2] + 1), dict(top_k=AT[3] + 2), dict(top_p=AT[4] + 2), dict(min_p=AT[5] + 2), dict(tokens=None),
                                    dict(tokens=AT[6] + 2), dict(shares=AT[7] + 1), dict(rows=-1), dict(vocabulary=0), dict(f32=2), dict(softcap=-1.0),
                                    dict(softcap=float("nan")), dict(softcap=float("inf")), dict(stride=-1), dict(stride=1 << 38),
                                    dict(tokens=AT[0] + 4 * 299), dict(shares=AT[1] + 8), dict(tokens=AT[7]), dict(shares=AT[3] - 8)])
def test_sample(lib, change):
    assert sample(lib, **change) == BAD


def test_more_than_a_row_or_a_grid_has(lib):
    assert sample(lib, vocabulary=step.MAX_VOCABULARY + 1) == TOO_LARGE and sample(lib, rows=1 << 27, stride=0) == TOO_LARGE


def test_calls_without_arguments(lib):
    for function in (lib.gevva_step_plan, lib.gevva_step_trim, lib.gevva_step_append, lib.gevva_step_sample):
        assert function(None, None) == BAD
    assert lib.gevva_moe_strerror(-8).decode().startswith("too few pages")


def test_packed_arguments_have_the_layout_of_the_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "gevva_moe.h"\nint main(void) {' + "".join(
        f'printf("%zu\\n", sizeof(gevva_step_{n}_args));' for n in ("plan", "trim", "append", "sample")) + "return 0; }")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "sizes"), str(source)], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [step._PLAN.size, step._TRIM.size, step._APPEND_AT.size, step._SAMPLE.size]


def test_every_declared_call_is_exported():
    lib = step._lib()
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gevva_moe.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(gevva_step_[a-z0-9_]+)\s*\(", text)))
    assert names == ["gevva_step_append", "gevva_step_plan", "gevva_step_sample", "gevva_step_trim"]
    for name in names:
        assert hasattr(lib, name)


class Pool:
    device = torch.device("cuda:0")


def test_python_mirror_refuses():
    ints, rows = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        step.PagePool(ints)
    with pytest.raises(ValueError, match="lengths"):
        step.plan_step(ints, ints, ints.view(3, 1), Pool, 16, 3)
    with pytest.raises(ValueError, match="lengths"):
        step.trim_step(ints, ints, ints.view(3, 1), Pool, 16)
    with pytest.raises(ValueError, match="CUDA"):
        step.kv_append_at(rows, rows, rows, None, ints, ints, None)
    for logits in (torch.zeros(2, 5), torch.zeros(2, 5, dtype=torch.float16), torch.zeros(5)):
        with pytest.raises(ValueError, match="logits"):
            step.sample_tokens(logits, torch.zeros(2))


def test_peers_are_touched_behind_a_cluster_barrier():
    """In the kernels that are launched in clusters a peer's shared memory is touched when all CTAs have begun: behind the first wait for the cluster."""
    csrc = os.path.join(ROOT, "gevva_b200", "csrc")
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(csrc, "sample.cu")).read(), flags=re.S)
    kernel = text[text.index("__global__"):]
    wait = kernel.index("cluster_wait()")
    assert kernel.index("cluster_arrive()") < wait
    for remote in ("cluster_map_shared(", "gather<T", "cluster_sums<", "window_of_bins<", "border_from_list<", "locate<T", "find_border<T", "sum_listed<T"):
        assert kernel.index(remote) > wait, remote
    pages = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(csrc, "step_pages.cu")).read(), flags=re.S)
    assert "cluster_map_shared" not in pages and pages.index("cluster_sync_all()") < pages.index("p.lengths_out[s]")
