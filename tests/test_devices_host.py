"""The entry points on the devices of one process: the library's objects linked against a runtime of two
devices that launches nothing but keeps their shared-memory limits apart (fake_cudart.cpp)."""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import sys
import textwrap

import pytest

from conftest import ROOT

CUDA = pathlib.Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"
HERE = pathlib.Path(__file__).resolve().parent

CALLS = '''
import ctypes, os, sys
from qwen_mla_vllm_b200 import _lib
lib = _lib.load()
P = 1 << 20  # an aligned address that nothing reads


def packed(cls, **kw):
    p = cls()
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def cache(dev, fp8=False):
    return dict(kv_cache=P, kv_stride_page=16 * 1024, kv_stride_token=1024, kv_row_width=1024, kv_dtype=3 if fp8 else 0,
                page_size=16, block_table=P, block_table_stride=4096, rms_offset=1000, rms_mode=3 if fp8 else 1,
                rank=768, qk_dim=1000, num_heads=24, sm_scale=0.1, q=P, q_pe=P + 2048, q_stride_row=24000, q_stride_head=1000,
                qpe_stride_row=24000, qpe_stride_head=1000, workspace=P, workspace_bytes=1 << 40, device=dev)


def tree(dev, **kw):
    d = dict(cache(dev, kw.pop("fp8", False)), kv_num_pages=4096, block_table_cols=4096, ctx_lens=P, tree_mask=P, num_reqs=4,
             num_nodes=8, o=P, o_stride_row=24 * 768, o_stride_head=768, lse=P, lse_stride_row=24, lse_dtype=2)
    p = packed(_lib.TreeParams, **dict(d, **kw))
    return lib.qmla_tree_attention(ctypes.addressof(p), None)


def tree_size(dev):
    p = packed(_lib.TreeParams, **cache(dev), kv_num_pages=4096, block_table_cols=4096, num_reqs=4, num_nodes=8)
    n = ctypes.c_int64()
    return lib.qmla_tree_workspace_bytes(ctypes.addressof(p), ctypes.byref(n)), n.value


def generic(dev, fp8=False):  # rank 1792 is the CUDA-core kernel's, with 64 KB of queries
    return tree(dev, fp8=fp8, rank=1792, qk_dim=2024, rms_offset=2024, kv_row_width=2048, kv_stride_token=2048, kv_stride_page=16 * 2048)


def weights(dev, fp8=False):
    p = packed(_lib.WeightsParams, **cache(dev, fp8), kv_num_pages=4096, block_table_cols=4096, seq_lens=P, num_reqs=4, qrows=1,
               lse=P, lse_stride_row=24, weights=P, weights_stride_req=65536, weights_cols=65536, decay=1.0)
    return lib.qmla_accumulate_weights(ctypes.addressof(p), None)


def evict(dev):
    p = packed(_lib.EvictParams, kv_cache=P, page_stride_bytes=1 << 15, token_stride_bytes=2048, row_bytes=2048, kv_num_pages=1 << 16,
               page_size=16, block_table=P, block_table_stride=1 << 14, block_table_cols=1 << 14, weights=P, positions=P, cols=250000,
               weights_stride_req=250000, positions_stride_req=250000, seq_lens=P, budget=1000, new_weights=P, new_positions=P,
               new_stride_req=1000, new_cols=1000, new_lens=P, num_reqs=2, workspace=P, workspace_bytes=1 << 40, device=dev)
    return lib.qmla_evict(ctypes.addressof(p), None)


def update(dev, fp8=False):
    p = packed(_lib.RopeCacheParams, q_pe=P, q_out=P, q_stride_token=24 * 8192, q_stride_head=8192, q_out_stride_token=24 * 8192,
               q_out_stride_head=8192, latent=P, latent_stride=768, k_pe=P, k_pe_stride=8224, positions=P, slot_mapping=P, steps=P,
               kv_cache=P, kv_stride_page=16 * 9216, kv_stride_token=9216, num_tokens=1000, num_pages=64, page_size=16,
               kv_row_width=9216, kv_dtype=3 if fp8 else 0, num_heads=24, rank=768, rope_width=8192, rot_dim=64, rms_heads=24,
               rms_mode=3 if fp8 else 1, scale=1.0, k_scale=P, device=dev)
    return lib.qmla_rope_cache_write(ctypes.addressof(p), None)


def calls(dev):
    for fp8 in (False, True):
        for f in (tree, generic, weights, update):
            before = lib.fake_launches(dev)
            assert f(dev, fp8=fp8) == 0, (f.__name__, fp8, dev)
            assert lib.fake_launches(dev) > before
    assert evict(dev) == 0
    assert lib.fake_current() == 0 and lib.fake_refused() == 0
'''

DECODE_CALLS = '''
def decode(dev, fp8=False):
    d = cache(dev, fp8)
    p = packed(_lib.DecodeParams, **d, kv_num_pages=4096, seq_lens=P, num_rows=4, qrows=1, o=P, o_stride_row=24 * 768, o_stride_head=768,
               lse=P, lse_stride_row=24, lse_dtype=2)
    return lib.qmla_mla_decode(ctypes.byref(p), None)


def gather(dev, fp8=False):
    p = packed(_lib.GatherParams, src_cache=P, src_stride_page=16 * 1024, src_stride_token=1024, page_size=16, num_pages=64,
               src_dtype=3 if fp8 else 0, row_elems=1024, rms_offset=1000, rms_heads=24, rms_mode=3, scale=P, block_table=P,
               block_table_stride=64, block_table_cols=64, cu_seq_lens=P, token_to_seq=P, num_seqs=2, num_tokens=5000, dst=P,
               dst_stride_row=1024, device=dev)
    return lib.qmla_gather_cache(ctypes.byref(p), None)


for dev in ORDER:
    for fp8 in (False, True):
        for f in (decode, gather):
            before = lib.fake_launches(dev)
            assert f(dev, fp8=fp8) == 0, (f.__name__, fp8, dev)
            assert lib.fake_launches(dev) > before
assert lib.fake_current() == 0 and lib.fake_refused() == 0
'''

SCRIPTS = {
    "the current device first": "calls(0); calls(1)",
    "another device first": "calls(1); calls(0)",
    "sizes asked for another device": "assert tree_size(1)[0] == 0; calls(1)",
    # the tensor-core kernel's scratch is not the other's: a query that failed once must not choose for good
    "a query that fails is asked again": """
        lib.fake_fail_queries(1)
        assert tree_size(0) == (-5, 0)  # the device's attributes
        assert weights(0) == 0          # known now, and nothing is left of the failure
        lib.fake_fail_queries(1)
        assert tree_size(0) == (-5, 0)  # the kernel's occupancy
        rc, n = tree_size(0)
        assert rc == 0 and n > 1 << 24, (rc, n)
        assert tree_size(1) == (0, n)
        calls(0); calls(1)
    """,
}


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    if shutil.which("g++") is None or not (CUDA / "cuda_runtime_api.h").exists():
        pytest.skip("needs g++ and the CUDA headers")
    from qwen_mla_vllm_b200 import build
    build.build()
    objs = sorted(build.OBJ.glob("*.o"))
    if not objs:
        pytest.skip("the library was built elsewhere: no objects to link")
    out = tmp_path_factory.mktemp("fake") / "libqmla_fake.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-w", f"-I{CUDA}", "-o", str(out), str(HERE / "fake_cudart.cpp"),
                    *map(str, objs), "-Wl,-Bsymbolic"], check=True)
    return out


def check(lib, script):
    env = dict(os.environ, QMLA_LIB_PATH=str(lib), PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", CALLS + script], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("name", SCRIPTS)
def test_two_devices(fake_lib, name):
    check(fake_lib, textwrap.dedent(SCRIPTS[name]))


@pytest.mark.parametrize("order", ["(0, 1)", "(1, 0)"])
def test_decode_and_gather_on_two_devices(fake_lib, order):
    check(fake_lib, f"ORDER = {order}\n" + DECODE_CALLS)
