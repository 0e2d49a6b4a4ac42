"""The paged 8-bit KV cache without a GPU: refusals, C structures, and the oracle against hand-made cases."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

import fa_b200
from fa_b200 import _lib
from oracle import paged_cache_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4M3 = torch.float8_e4m3fn


def cache_args(blocks=4, bs=16, heads=2, dim=64, dtype=E4M3):
    c = lambda: torch.zeros(blocks, bs, heads, dim, dtype=torch.int8).view(dtype)
    return [c(), c(), torch.ones(blocks, heads), torch.ones(blocks, heads)]


def decode_args(**kw):
    c = cache_args(**kw)
    dim, heads = c[0].shape[3], c[0].shape[2]
    return [torch.zeros(3, 2 * heads, dim, dtype=torch.float16), *c, torch.zeros(3, 2, dtype=torch.int32),
            torch.zeros(3, dtype=torch.int32)]


def append_args(tokens=5, **kw):
    c = cache_args(**kw)
    x = torch.zeros(tokens, c[0].shape[2], c[0].shape[3], dtype=torch.bfloat16)
    return [x, x.clone(), *c, torch.zeros(tokens, dtype=torch.int64)]


def plan_args(batch=3):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    return [i(batch), i(batch), i(batch, 4), i(9), i(1), 6, 16]


def with_(args, **changes):
    args = list(args)
    for k, v in changes.items():
        args[int(k[1:])] = v
    return args


ODD_STRIDE = torch.zeros(4, 16, 2, 72, dtype=torch.int8)[..., :64]


@pytest.mark.parametrize("change, message", [
    (dict(_0=torch.zeros(3, 4, 64)), "float16 or bfloat16"),
    (dict(_0=torch.zeros(3, 64, dtype=torch.float16)), "batch, heads, dim"),
    (dict(_0=torch.zeros(3, 3, 64, dtype=torch.float16)), "multiple of cache heads"),
    (dict(_0=torch.zeros(3, 4, 128, dtype=torch.float16)), "head_dim must match"),
    (dict(_1=torch.zeros(4, 16, 2, 64, dtype=torch.float16)), "float8_e4m3fn or int8"),
    (dict(_1=torch.zeros(4, 16, 2, 64, dtype=torch.int8)), "same shape and dtype"),
    (dict(_2=torch.zeros(5, 16, 2, 64, dtype=torch.int8).view(E4M3)), "same shape and dtype"),
    (dict(_1=ODD_STRIDE.view(E4M3), _2=ODD_STRIDE.view(E4M3)), "rows aligned to 16 bytes"),
    (dict(_1=torch.zeros(4, 16, 1, 64, dtype=torch.int8).view(E4M3).expand(4, 16, 2, 64)), "broadcast"),
    (dict(_3=torch.ones(4, 2, dtype=torch.float16)), "float32"),
    (dict(_3=torch.ones(4, 3)), "shape"),
    (dict(_5=torch.zeros(3, 2, dtype=torch.int64)), "int32"),
    (dict(_5=torch.zeros(2, 2, dtype=torch.int32)), "invalid shape"),
    (dict(_5=torch.zeros(3, 0, dtype=torch.int32)), "at least one"),
    (dict(_6=torch.zeros(3, 1, dtype=torch.int32)), "invalid shape"),
])
def test_decode_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        fa_b200.flash_attention_decode_paged_8bit(*with_(decode_args(), **change))


@pytest.mark.parametrize("kw, message", [(dict(bs=12), "power of two"), (dict(dim=48), "head_dim"),
                                         (dict(dim=512), "head_dim"), (dict(blocks=0), "positive")])
def test_cache_shape_refusals(kw, message):
    with pytest.raises(ValueError, match=message):
        fa_b200.flash_attention_decode_paged_8bit(*decode_args(**kw))
    with pytest.raises(ValueError, match=message):
        fa_b200.paged_kv_append(*append_args(**kw))


@pytest.mark.parametrize("change, message", [
    (dict(_0=torch.zeros(5, 2, 64)), "float16 or bfloat16"),
    (dict(_1=torch.zeros(5, 2, 64, dtype=torch.float16)), "share"),
    (dict(_1=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "same shape"),
    (dict(_0=torch.zeros(5, 4, 64, dtype=torch.bfloat16), _1=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), "same heads"),
    (dict(_4=torch.ones(4, 1).expand(4, 2)), "broadcast"),
    (dict(_6=torch.zeros(5, dtype=torch.int32)), "int64"),
    (dict(_6=torch.zeros(6, dtype=torch.int64)), "one entry"),
])
def test_append_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        fa_b200.paged_kv_append(*with_(append_args(), **change))


@pytest.mark.parametrize("change, message", [
    (dict(_0=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(_1=torch.zeros(4, dtype=torch.int32)), "same batch size"),
    (dict(_2=torch.zeros(3, 0, dtype=torch.int32)), "at least one"),
    (dict(_2=torch.zeros(4, 3, dtype=torch.int32).T), "unit inner stride"),
    (dict(_2=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), "overlap"),
    (dict(_3=torch.zeros(18, dtype=torch.int32)[::2]), "contiguous"),
    (dict(_4=torch.zeros(2, dtype=torch.int32)), "one element"),
    (dict(_5=-1), "num_tokens"), (dict(_5=2 ** 31), "num_tokens"), (dict(_5=True), "num_tokens"),
    (dict(_6=12), "power of two"), (dict(_6=2 ** 30), "fewer than"),
])
def test_plan_refusals(change, message):
    with pytest.raises(ValueError, match=message):
        fa_b200.paged_kv_plan(*with_(plan_args(), **change))


def test_other_refusals():
    with pytest.raises(ValueError, match="requests"):
        fa_b200.paged_kv_plan(*plan_args(8193))
    with pytest.raises(ValueError, match="updated in place"):
        fa_b200.paged_kv_plan(*with_(plan_args(), _0=torch.zeros(6, dtype=torch.int32)[::2]), inplace=True)
    with pytest.raises(TypeError, match="slot_mapping"):
        fa_b200.paged_kv_append(*append_args()[:6], None)
    for bad in (dict(layers=0), dict(dtype=torch.float16), dict(max_batch=2.0)):
        kw = dict(layers=1, num_blocks=4, block_size=16, kv_heads=2, head_dim=64, max_batch=2, max_blocks=2, device="cpu")
        with pytest.raises(ValueError):
            fa_b200.PagedKVCache8(**{**kw, **bad})
    if not torch.cuda.is_available():   # the platform is asked last, after every contract
        for call, args in ((fa_b200.flash_attention_decode_paged_8bit, decode_args()),
                           (fa_b200.paged_kv_append, append_args()), (fa_b200.paged_kv_plan, plan_args())):
            with pytest.raises(RuntimeError, match="requires"):
                call(*args)


@pytest.mark.parametrize("index", range(5))
def test_inference_only_whatever_needs_the_gradient(monkeypatch, index):
    """Scales (and e4m3 caches) are floating tensors too: no gradient would reach them, so the calls refuse."""
    from fa_b200 import _validation

    monkeypatch.setattr(_validation, "_require_platform", lambda device: None)
    args = decode_args()
    args[index].requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference-only"):
        fa_b200.flash_attention_decode_paged_8bit(*args)
    args = append_args()
    args[index + 1].requires_grad_(True)            # value, caches, scales
    with pytest.raises(RuntimeError, match="inference-only"):
        fa_b200.paged_kv_append(*args)


def test_c_entries_refuse_without_a_gpu():
    lib = _lib.load()
    for fn, cls in ((lib.fa_paged_plan, _lib.PagedPlanParams), (lib.fa_paged8_append, _lib.Paged8AppendParams),
                    (lib.fa_decode_paged8, _lib.Paged8Params)):
        assert fn(None, None) == -1
    assert lib.fa_paged_plan(ctypes.byref(_lib.PagedPlanParams()), None) == -1
    assert lib.fa_paged8_append(ctypes.byref(_lib.Paged8AppendParams()), None) == 0        # no tokens, nothing to do
    assert lib.fa_paged8_append(ctypes.byref(_lib.Paged8AppendParams(num_tokens=1)), None) == -1
    assert lib.fa_decode_paged8(ctypes.byref(_lib.Paged8Params()), None) == -1
    assert lib.fa_decode_paged8(ctypes.byref(_lib.Paged8Params(batch=1, heads_q=1, max_blocks=1)), None) == -1
    x = torch.zeros(64, dtype=torch.uint8)
    at = x.data_ptr() - x.data_ptr() % 16 + 16
    plan = dict(batch=2, max_blocks=4, num_blocks=4, block_size=16, num_tokens=1, context_lens=at, new_lens=at,
                block_table=at, bt_stride=4, free_blocks=at, free_count=at, slot_mapping=at, cu_seqlens=at,
                context_lens_out=at, free_count_out=at)
    for bad in (dict(block_size=3), dict(batch=8193), dict(bt_stride=3), dict(free_count=None), dict(num_tokens=-1)):
        assert lib.fa_paged_plan(ctypes.byref(_lib.PagedPlanParams(**{**plan, **bad})), None) < 0, bad
    strides = (2048, 128, 64, 1)
    append = dict(dtype=_lib.FA_F16, cache_dtype=0, heads_kv=2, head_dim=64, num_blocks=4, block_size=16, num_tokens=1,
                  key=at, key_strides=(128, 64, 1), value=at, value_strides=(128, 64, 1), k_cache=at, k_strides=strides,
                  v_cache=at, v_strides=strides, k_scales=at, v_scales=at, slot_mapping=at)
    for bad in (dict(dtype=_lib.FA_F32), dict(cache_dtype=2), dict(head_dim=72), dict(head_dim=96), dict(head_dim=512), dict(block_size=24),
                dict(k_cache=at + 8), dict(v_strides=(2048, 128, 64, 2)), dict(k_strides=(2048, 128, 72, 1)),
                dict(k_strides=(0, 128, 64, 1)), dict(key=at + 8), dict(key_strides=(128, 60, 1)), dict(v_scales=None)):
        assert lib.fa_paged8_append(ctypes.byref(_lib.Paged8AppendParams(**{**append, **bad})), None) < 0, bad


def test_c_plan_refuses_strided_lengths_in_place():
    """The kernel reads context_lens with its stride and writes context_lens_out densely: as one tensor they need stride 1."""
    lib = _lib.load()
    x = (ctypes.c_int64 * 64)()
    at, other = ctypes.addressof(x), ctypes.addressof(x) + 256
    plan = dict(batch=2, max_blocks=4, num_blocks=4, block_size=16, num_tokens=1, context_lens=at, new_lens=at, nl_stride=1,
                block_table=at, bt_stride=4, free_blocks=at, free_count=at, slot_mapping=at, cu_seqlens=at,
                free_count_out=at)
    assert lib.fa_paged_plan(ctypes.byref(_lib.PagedPlanParams(**plan, cl_stride=2, context_lens_out=at)), None) == -1
    assert b"contiguous" in lib.fa_last_error_string()
    if not torch.cuda.is_available():               # (addresses of host memory: nothing is launched without a device)
        for kw in (dict(cl_stride=2, context_lens_out=other), dict(cl_stride=1, context_lens_out=at)):
            assert lib.fa_paged_plan(ctypes.byref(_lib.PagedPlanParams(**plan, **kw)), None) != -1


def build_module():
    import importlib.util

    path = os.path.join(ROOT, "flash-attention-rdna3_b200", "build.py")
    spec = importlib.util.spec_from_file_location("fa_b200_build_module", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_library_builds_without_torch(monkeypatch, capsys, tmp_path):
    """Only the Python binding needs PyTorch: without it the build ends with the library and says so."""
    import sys

    build = build_module()
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "binding.so"))
    monkeypatch.setitem(sys.modules, "torch", None)                 # import torch raises ImportError
    assert build.build() == build.OUT
    assert "not built" in capsys.readouterr().err and not os.path.exists(build.BINDING)
    monkeypatch.setattr(build, "_build_binding", lambda *a: pytest.fail("built"))
    assert build.build(binding=False) == build.OUT


def test_the_binding_is_built_again_for_another_torch(monkeypatch):
    build = build_module()
    build.build()
    ran = []

    def compiler(cmd, **kw):
        ran.append(cmd)
        return subprocess.CompletedProcess(cmd, 1, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build()                                                   # all is up to date
    assert not ran
    monkeypatch.setattr(torch, "__version__", "2.8.0")
    with pytest.raises(RuntimeError, match="no-binding"):
        build.build()
    assert len(ran) == 1 and '-DFA_TORCH="2.8.0"' in ran[0]


def test_a_binding_of_another_torch_is_refused(monkeypatch):
    module = _lib.paged_binding()
    _lib._check_binding(module)
    monkeypatch.setattr(torch, "__version__", "2.8.0")
    with pytest.raises(RuntimeError, match="built for PyTorch"):
        _lib._check_binding(module)


def test_struct_sizes_match_the_header():
    src = ('#include "fa_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){'
           'printf("%zu %zu %zu %zu %zu %d %d", sizeof(fa_paged_plan_params), sizeof(fa_paged8_append_params), '
           'sizeof(fa_paged8_params), offsetof(fa_paged8_params, softmax_scale), '
           'offsetof(fa_paged8_append_params, slot_mapping), FA_PLAN_MAX_BATCH, FA_STATUS_SLOT_ORDER);return 0;}\n')
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "s.c"), "-o", os.path.join(d, "s")],
                       check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.PagedPlanParams), ctypes.sizeof(_lib.Paged8AppendParams),
                   ctypes.sizeof(_lib.Paged8Params), _lib.Paged8Params.softmax_scale.offset,
                   _lib.Paged8AppendParams.slot_mapping.offset, _lib.FA_PLAN_MAX_BATCH, _lib.FA_STATUS_SLOT_ORDER]


def test_oracle_plan_by_hand():
    """Two pages of 4: request 0 grows into a new page, request 1 ends and returns its pages, request 2 finds none left."""
    table = torch.tensor([[7, -1], [3, 5], [-1, -1]], dtype=torch.int32)
    stack = torch.tensor([9, 0, 0, 0], dtype=torch.int32)
    slots, cu, lens, count, table2, stack2 = oracle.plan_ref([4, 8, 0], [2, -1, 8], table, stack, 1, 10, 4)
    assert lens == [6, 0, 8] and cu == [0, 2, 2, 10] and count == 0
    assert table2 == [[7, 5], [3, 5], [3, 9]]
    assert stack2 == [9, 0, 0, 0]
    assert slots[:2] == [-1, -1]            # page 5 lies outside a pool of 4 pages
    assert slots[2:6] == [12, 13, 14, 15] and slots[6:] == [-1] * 4
    _, _, lens, count, _, stack3 = oracle.plan_ref([4, 8, 0], [2, -1, 9], table, stack, 1, 11, 4)
    assert lens == [6, 0, 0] and count == 2 and stack3 == [9, 3, 0, 0]


def test_oracle_codes_agree_with_torch():
    """The oracle's e4m3 rounding against torch's cast, over every representable value and the midpoints between them."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat((codes, mid, mid * (1 + 1e-12), mid * (1 - 1e-12), torch.tensor([500.0, 447.0], dtype=torch.float64)))
    x = torch.cat((x, -x))
    want = x.clamp(-448, 448)
    near = (want[:, None] - torch.cat((codes, -codes))[None]).abs().amin(1)
    got = oracle.round_codes(x, E4M3)
    assert torch.equal((got - want).abs(), near)
    exact = torch.cat((codes, mid))
    assert torch.equal(oracle.round_codes(exact, E4M3), exact.float().to(E4M3).double())    # ties to even
    assert oracle.scale_for(torch.tensor([448.0, 448.5, 0.0], dtype=torch.float64), E4M3).tolist() == [1.0, 2.0, 2.0 ** -126]
    assert oracle.scale_for(torch.tensor([127.0, 127.5], dtype=torch.float64), torch.int8).tolist() == [1.0, 2.0]


def test_oracle_append_rounds_a_grown_page_again():
    cache = torch.zeros(1, 4, 1, 16, dtype=torch.int8)
    cache[0, 0] = 3
    x = torch.full((1, 1, 16), 200.0, dtype=torch.float16)
    codes, scales = oracle.append_ref(x, cache, torch.ones(1, 1), torch.tensor([1]))
    assert scales.item() == 2.0 and codes[0, 0].unique().tolist() == [2.0] and codes[0, 1].unique().tolist() == [100.0]
