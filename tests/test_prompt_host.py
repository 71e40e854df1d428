"""Refusals of the packed prompts and of the scoring head that need no GPU, and
(marked gpu) those that need a handle."""
from __future__ import annotations

import ctypes as C

import pytest


def test_prompt_defaults_and_bad_configs(vxk):
    lib = vxk.load()
    c = lib.vxk_prompt_default_config()
    assert c.struct_size == C.sizeof(vxk.PromptConfig)
    assert (c.n_q_heads, c.n_kv_heads, c.head_dim, c.dtype, c.causal, c.window) == (32, 8, 128, vxk.DTYPE_F16, 1, 0)
    h = C.c_void_p()
    for field, value in (("struct_size", 8), ("head_dim", 96), ("n_q_heads", 30), ("n_kv_heads", 0), ("max_seqs", 0),
                         ("max_rows", 0), ("max_position", -1), ("dtype", 0), ("dtype", 8), ("rope_theta", 0.0),
                         ("rope_theta", float("nan")), ("scale", -1.0), ("scale", float("inf")), ("causal", 2),
                         ("window", -1)):
        c = lib.vxk_prompt_default_config()
        setattr(c, field, value)
        assert lib.vxk_prompt_create(C.byref(c), C.byref(h)) == vxk.INVALID_ARGUMENT, field
        assert not h.value
        buf = C.create_string_buffer(256)
        assert lib.vxk_prompt_last_error(None, buf, 256) == vxk.OK and buf.value
    c = lib.vxk_prompt_default_config()
    c.causal, c.window = 0, 5  # a window looks back
    assert lib.vxk_prompt_create(C.byref(c), C.byref(h)) == vxk.INVALID_ARGUMENT
    assert lib.vxk_prompt_create(None, C.byref(h)) == vxk.INVALID_ARGUMENT


def test_null_handles(vxk):
    lib = vxk.load()
    n = C.c_int32()
    assert lib.vxk_prompt_plan(None, None, None, 1, None) == vxk.INVALID_ARGUMENT
    assert lib.vxk_prompt_rows(None, C.byref(n)) == vxk.INVALID_ARGUMENT
    assert lib.vxk_prompt_rope(None, *[None] * 7) == vxk.INVALID_ARGUMENT
    assert lib.vxk_prompt_attention(None, *[None] * 5) == vxk.INVALID_ARGUMENT
    assert lib.vxk_prompt_sync(None, None, 1) == vxk.INVALID_ARGUMENT
    lib.vxk_prompt_destroy(None)
    assert lib.vxk_head_score(None, None, None, 1, None, 0, *[None] * 5) == vxk.INVALID_ARGUMENT
    assert lib.vxk_head_score_logits(None, None, 0, 1, 1, None, 0, *[None] * 5) == vxk.INVALID_ARGUMENT


@pytest.mark.gpu
def test_prompt_call_refusals(vxk):
    import torch

    prompt = vxk.Prompt(n_q_heads=2, n_kv_heads=1, head_dim=64, max_seqs=3, max_rows=50, max_position=40)
    x = torch.zeros(50 * 2 * 64 + 8, device="cuda")
    a = x.data_ptr()

    def status(call, *args):
        with pytest.raises(vxk.VxkError) as e:
            call(*args)
        return e.value.status

    assert status(prompt.attention, a, a, a, a) == vxk.INVALID_STATE  # no plan yet
    assert status(prompt.plan, []) == vxk.INVALID_ARGUMENT
    assert status(prompt.plan, [1, 1, 1, 1]) == vxk.INVALID_ARGUMENT
    assert status(prompt.plan, [-1]) == vxk.INVALID_ARGUMENT
    assert status(prompt.plan, [30, 21]) == vxk.INVALID_ARGUMENT      # more than max_rows
    assert status(prompt.plan, [2 ** 31 - 1] * 3) == vxk.INVALID_ARGUMENT
    assert status(prompt.plan, [10], [31]) == vxk.INVALID_ARGUMENT    # reaches position 40
    assert status(prompt.plan, [10], [-1]) == vxk.INVALID_ARGUMENT
    assert status(prompt.plan, [10, 3], [2]) == vxk.INVALID_ARGUMENT
    assert prompt.plan([10, 0], [30, 1000]) == 10                     # a sequence without rows has no position
    assert status(prompt.attention, a, 0, a, a) == vxk.INVALID_ARGUMENT
    assert status(prompt.attention, a, a + 8, a, a) == vxk.INVALID_ARGUMENT
    assert status(prompt.rope, a, a, a, a, 0, a) == vxk.INVALID_ARGUMENT
    prompt.close()
    bare = vxk.Prompt(n_q_heads=2, n_kv_heads=1, head_dim=64, max_position=0)
    bare.plan([4])
    assert status(bare.rope, a, a, a, a, a, a) == vxk.INVALID_STATE
    bare.close()


@pytest.mark.gpu
def test_score_call_refusals(vxk):
    import torch

    head = vxk.Head(dim=64, vocab=10)
    a = torch.zeros(4096, device="cuda").data_ptr()

    def refused(call, *args):
        with pytest.raises(vxk.VxkError) as e:
            call(*args)
        assert e.value.status == vxk.INVALID_ARGUMENT

    refused(head.score_logits, 0, 0, 10, 1, a, 0, a, a, a, a)
    refused(head.score_logits, a, 8, 10, 1, a, 0, a, a, a, a)       # type
    refused(head.score_logits, a, 0, 9, 1, a, 0, a, a, a, a)        # ld below vocab
    refused(head.score_logits, a + 2, 0, 10, 1, a, 0, a, a, a, a)   # not aligned to an element
    refused(head.score_logits, a, 0, 10, 0, a, 0, a, a, a, a)
    refused(head.score_logits, a, 0, 10, 1, a, 11, a, a, a, a)      # more than vocab
    refused(head.score_logits, a, 0, 10, 1, a, -1, a, a, a, a)
    refused(head.score_logits, a, 0, 10, 1, 0, 0, a, a, a, a)       # a log probability of no token
    refused(head.score, 0, a, 1, a, 0, a, a, a, a)
    refused(head.score, a, 0, 1, a, 0, a, a, a, a)
    refused(head.score, a + 8, a, 1, a, 0, a, a, a, a)
    refused(head.score, a, a + 4, 1, a, 0, a, a, a, a)
    refused(head.score, a, a, 1, a, 17, a, a, a, a)
    head.close()


def test_prompt_config_layout_matches_the_c_compiler(vxk, tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    names = [f[0] for f in vxk.PromptConfig._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include <vxk.h>\nint main(void) {\n"
                   + '    printf("%zu\\n", sizeof(vxk_prompt_config));\n'
                   + "".join(f'    printf("%zu\\n", offsetof(vxk_prompt_config, {n}));\n' for n in names) + "    return 0;\n}\n")
    exe = tmp_path / "layout"
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-I", str(include), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(vxk.PromptConfig)] + [getattr(vxk.PromptConfig, n).offset for n in names]
