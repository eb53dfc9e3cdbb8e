"""libcascade_lm.so loads and exports exactly what include/cascade_lm.h declares, and refuses bad calls. No GPU needed."""
import ctypes as C
import os
import re
import subprocess

from cascade_amd import _native_lm as native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_functions():
    src = open(os.path.join(ROOT, "include", "cascade_lm.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(csa_lm_[a-z0-9_]+)\s*\(", src)))


def test_header_and_binding_agree():
    assert declared_functions() == sorted(native.EXPORTS)


def test_library_exports_every_declared_symbol():
    lib = native.load()
    for name in declared_functions():
        assert hasattr(lib, name), name


def test_struct_layouts_match_the_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text('''#include <stddef.h>
#include <stdio.h>
#include "cascade_lm.h"
int main(void) {
    printf("%zu %zu %zu %zu %zu\\n", sizeof(csa_lm_attention), offsetof(csa_lm_attention, tokens), offsetof(csa_lm_attention, d_slope),
           offsetof(csa_lm_attention, cap), offsetof(csa_lm_attention, v));
    printf("%zu %zu\\n", sizeof(csa_lm_heads), offsetof(csa_lm_heads, head_stride));
    printf("%zu %zu %zu\\n", sizeof(csa_lm_values), offsetof(csa_lm_values, n), offsetof(csa_lm_values, type));
    return 0;
}
''')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    at, h, v = native.CsaLmAttention, native.CsaLmHeads, native.CsaLmValues
    assert [int(x) for x in lines[0].split()] == [C.sizeof(at), at.tokens.offset, at.d_slope.offset, at.cap.offset, at.v.offset]
    assert [int(x) for x in lines[1].split()] == [C.sizeof(h), h.head_stride.offset]
    assert [int(x) for x in lines[2].split()] == [C.sizeof(v), v.n.offset, v.type.offset]


def test_argument_errors_need_no_gpu():
    lib = native.load()
    bad, large = -1, -2
    work = C.create_string_buffer(64)
    assert lib.csa_lm_spans_u16_dev(None, 5, 0xFFFF, None, None, None, None, 0, None) == bad
    assert lib.csa_lm_spans_u16_dev(None, 5, 0x10000, None, None, None, None, 0, None) == bad
    assert lib.csa_lm_spans_u16_dev(None, 1 << 31, 0xFFFF, None, None, None, None, 0, None) == large
    assert lib.csa_lm_spans_u16_dev(None, 0, 0xFFFF, None, None, None, None, 0, None) == 0
    assert lib.csa_lm_attention_forward_dev(None, native.CsaLmHeads(), None, None, 0, None) == bad
    assert b"null" in lib.csa_lm_last_error()
    assert lib.csa_lm_cross_entropy_forward_dev(0, None, 8, None, 8, None, 4, 8, 10, None, None, None, 0, None) == bad
    assert lib.csa_lm_cross_entropy_forward_dev(7, None, 8, None, 8, None, 4, 8, 10, None, None, None, 0, None) == bad
    assert lib.csa_lm_cross_entropy_forward_dev(0, None, 8, None, 8, None, 1 << 31, 8, 10, None, None, None, 0, None) == large
    assert lib.csa_lm_cross_entropy_forward_dev(0, None, 8, None, 8, None, 4, 0, 10, None, None, None, 0, None) == bad
    one = (native.CsaLmValues * 1)(native.CsaLmValues(C.addressof(work), C.addressof(work), 3, 9))
    assert lib.csa_lm_clip_dev(one, 1, 1.0, None, None, 0, None) == bad
    one[0].type = native.CSA_LM_F32
    assert lib.csa_lm_clip_dev(one, 1, -1.0, None, None, 0, None) == bad
    assert lib.csa_lm_clip_dev(one, 1, float("nan"), None, None, 0, None) == bad
    assert lib.csa_lm_clip_dev(one, 1, 1.0, None, None, 0, None) == bad and b"workspace" in lib.csa_lm_last_error()
    assert lib.csa_lm_clip_dev(None, 1, 1.0, None, None, 0, None) == bad


def test_workspace_sizes():
    lib = native.load()
    assert lib.csa_lm_spans_workspace(4096) == 0 and lib.csa_lm_spans_workspace(4097) == 16384
    assert lib.csa_lm_cross_entropy_workspace(8, 0, 10, 0) == 0
    # attention: 16 bytes a row and head, and bounded sums, whatever the length and the heads
    for tokens in (1, 129, 4000, 16384, 131072, 1 << 20, 1 << 24):
        for heads, kv_heads in ((1, 1), (16, 16), (16, 2), (64, 8), (71, 1), (128, 1)):
            for flags, most in ((0, 80 << 20), (native.CSA_LM_BACKWARD, (700 << 20) + (tokens + 32) * heads * 16 + tokens // 4)):
                assert lib.csa_lm_attention_workspace(tokens, heads, kv_heads, 128, flags) <= most, (tokens, heads, kv_heads, flags)
    small, copies = (lib.csa_lm_cross_entropy_workspace(64, 512, 50257, f) for f in (0, native.CSA_LM_COPY_ROWS))
    assert copies - small >= 50257 * 512 * 2
    # the logits of a batch, or their gradients, are never all there: 8192 x 50257 values of 16 bits are 823 MB
    assert lib.csa_lm_cross_entropy_workspace(8192, 1024, 50257, native.CSA_LM_BACKWARD) < 400 << 20
    assert lib.csa_lm_cross_entropy_workspace(8192, 1024, 50257, 0) < 64 << 20
