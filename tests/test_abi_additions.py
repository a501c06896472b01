"""The entry points beyond the reference's headers, by name: each is exported, declared with what it adds, and bound in
device.py; where the reference tree is present, they are exactly what the library exports beyond its device.h."""
import os
import re
import subprocess

import pytest

from __graft_entry__ import ROOT, load_device

dev = load_device()
HEADER = os.path.join(ROOT, "include", "vibevoice_hip.h")
REF_HEADER = "/root/reference/include/vibevoice/device.h"

KV_QUANT = {"vv_kv_rotate_dev", "vv_kv_unrotate_dev"}        # the reference's kv_quant.h:96-101, which its decoder links against
ADDITIONS = {
    "vv_add_rmsnorm_dev", "vv_rope_qk_dev", "vv_bias_rope_qk_dev", "vv_embedding_rmsnorm_dev", "vv_gemv_multi_dev",
    "vv_gemv_swiglu_dev", "vv_attn_decode_static", "vv_rope_table_dev", "vv_gemm_bias_rope_dev", "vv_gemm_swiglu_dev",
    "vv_gemm_qkv_rope_dev", "vv_kv_page_plan_dev", "vv_rope_kv_append_dev", "vv_attn_decode_batch",
    "vv_attn_decode_batch_scratch_bytes"}


def exported():
    out = subprocess.check_output(["nm", "-D", "--defined-only", dev.LIB_PATH], text=True)
    return {line.split()[-1] for line in out.splitlines() if " T vv_" in line}


def test_additions_are_exported_and_bound():
    assert ADDITIONS | KV_QUANT <= exported()
    assert ADDITIONS | KV_QUANT <= set(dev.SIGNATURES)
    assert all(callable(getattr(dev, name)) for name in ADDITIONS)


def test_the_serving_additions_say_so_in_the_header():
    """The comment before each declaration: an addition, or the scratch of one."""
    text = open(HEADER).read()
    for name in ("vv_kv_page_plan_dev", "vv_rope_kv_append_dev", "vv_attn_decode_batch"):
        at = re.search(rf"^vv_status_t {name}\(", text, flags=re.M).start()
        comment = text[text.rfind("/*", 0, at):at]
        assert comment.startswith("/* addition:") and comment.rstrip().endswith("*/"), name
        assert "replaces device.h" not in comment


@pytest.mark.skipif(not os.path.exists(REF_HEADER), reason="reference tree not present")
def test_additions_are_all_there_is_beyond_the_reference():
    text = re.sub(r"/\*.*?\*/", "", open(REF_HEADER).read(), flags=re.S)
    wanted = set(re.findall(r"^\s*(?:vv_status_t|int|size_t|void|bool|const char\*)\s+(vv_[a-z0-9_]+)\s*\(",
                            text, flags=re.M))
    assert exported() - wanted == ADDITIONS | KV_QUANT
