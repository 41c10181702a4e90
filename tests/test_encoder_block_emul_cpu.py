"""The encoder block's GPU tests (tests/test_gpu_encoder_block.py) on the CPU build of their kernel files (tests/emul): the same functions, the host as the device, at
the sizes a fiber per work-item can walk; refusals of every entry point; the reference against torch's autograd."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

import encoder_block_reference as R  # noqa: E402
import test_gpu_encoder_block as T  # noqa: E402
from test_kernels_emul_cpu import HE, emulated_library  # noqa: E402,F401  (fixtures)

CPU = torch.device("cpu")
F32, BF16, F16 = T.F32, T.BF16, T.F16


@pytest.mark.parametrize("n,d,stream,kind,norm", [(3, 2, F32, F32, "RMS"), (5, 100, F32, F32, "LAYER"), (7, 257, BF16, BF16, "LAYER"), (2, 1000, F32, BF16, "RMS"), (3, 520, F32, F32, "LAYER"),
                                                  (2, 2047, F16, F16, "RMS"), (1, 4100, F32, F16, "RMS"), (2, 8192, BF16, BF16, "LAYER"), (1, 8191, F32, F32, "RMS")])
def test_emulated_residual_norm(HE, n, d, stream, kind, norm):
    T.test_residual_norm_both_ways(HE, CPU, n, d, stream, kind, norm)


def test_emulated_residual_norm_other_forms(HE):
    T.test_residual_norm_alone_strided_and_of_other_parameter_types(HE, CPU, BF16, "LAYER")
    T.test_residual_norm_rows_apart(HE, CPU)
    T.test_residual_norm_gradient_against_differences(HE, CPU)


@pytest.mark.parametrize("shape,heads,kv,dim,kind", [("one", 1, 1, 1, F32), ("none", 4, 4, 32, F32), ("ordinary", 4, 4, 25, F16), ("ordinary", 8, 2, 64, BF16), ("long", 6, 2, 33, F32),
                                                     ("first empty", 12, 1, 100, BF16), ("last empty", 65, 5, 7, F32), ("single entry", 1, 1, 256, F32)])
def test_emulated_neighbor_attention(HE, shape, heads, kv, dim, kind):
    T.test_neighbor_attention_both_ways(HE, CPU, shape, heads, kv, dim, kind)


@pytest.mark.parametrize("masked", [1, 6])
def test_emulated_neighbor_attention_masks(HE, masked):
    T.test_neighbor_attention_with_a_bias_that_masks(HE, CPU, masked, 8, 2, 64, BF16)
    T.test_neighbor_attention_lowest_value_and_masked_garbage(HE, CPU, F32)


def test_emulated_neighbor_attention_other_forms(HE):
    T.test_neighbor_attention_two_lists_and_own_rows(HE, CPU)
    T.test_neighbor_attention_gradient_against_differences(HE, CPU)
    T.test_neighbor_attention_hubs_strides_and_repeats(HE, CPU)


@pytest.mark.parametrize("bits,param,grad,sizes", [(32, F32, F32, [255, 256, 257]), (8, F32, F32, [0, 5, 0, 2048, 2049]), (8, BF16, F16, [3] * 70), (32, F16, BF16, [7, 8, 9, 1000]), (8, F32, F32, [1])])
def test_emulated_adamw(HE, bits, param, grad, sizes):
    T.test_adamw_step(HE, CPU, bits, param, grad, sizes)


def test_emulated_adamw_other_forms(HE):
    T.test_adamw_leaves_out_what_has_no_gradient_and_steps_by_a_device_counter(HE, CPU)


# ------------------------------------------------------------------------------------------------ refusals
def refused(HE, message, call, *a, **k):
    with pytest.raises(HE.MariusHipError, match=message):
        call(*a, **k)


def test_residual_norm_refuses(HE):
    x, w = torch.zeros(4, 8), torch.ones(8)
    f, b = HE.residual_norm, HE.residual_norm_backward
    refused(HE, "nothing to compute", f, x, pre_norm=False)
    refused(HE, "need a block", f, x, gate=w)
    refused(HE, "need a block", f, x, post_norm=True)
    refused(HE, "needs a block", f, x, residual_scale=0.5)
    refused(HE, "differ in shape", f, x, x[:, :4])
    refused(HE, "the block's type", f, x.half(), x)
    refused(HE, "the block's type", f, x.half(), x.bfloat16())
    refused(HE, "float32, bfloat16 or float16", f, x.double())
    refused(HE, "rows \\[n, d\\]", f, x[0])
    refused(HE, "kind is one of", f, x, kind="BATCH")
    refused(HE, "Unsupported activation", f, x, x, w, gate_activation="GELU")
    refused(HE, "rows have 8 elements", f, x, pre_weight=w[:4])
    refused(HE, "not there", f, x, x, post_weight=w)
    refused(HE, "of one type", f, x, x, pre_weight=w, pre_bias=w.half())
    refused(HE, "gate is", f, x, x, w[:3])
    refused(HE, "element gate", f, x, x, x.half())
    refused(HE, "1 to 8192", f, torch.zeros(1, 8193))
    refused(HE, "eps", f, x, eps=-1.0)
    refused(HE, "grad_h is not like h", b, x, x[:2], x)
    refused(HE, "grad_y is not like y", b, x.half(), x, x)
    refused(HE, "no gradient", b, None, None, x)
    refused(HE, "grad_h is not like h", b, x, x, x, x, pre_norm=False, post_norm=True)


def test_residual_norm_c_abi_refuses(HE):
    """the C entry points check what they are given themselves"""
    L, x = HE.lib(), torch.zeros(4, 8)
    m = HE.ResidualNorm(n=4, d=8, pre_norm=1, residual_scale=1.0)
    P = HE.ptr
    assert L.marius_residual_norm_forward(None, P(x), 8, None, 0, None, 0, P(x), 8, None) == 1
    assert L.marius_residual_norm_forward(C.byref(m), P(x), 7, None, 0, None, 0, P(x), 8, None) == 1
    assert L.marius_residual_norm_forward(C.byref(m), P(x), 8, None, 0, None, 0, None, 8, None) == 1
    for field, value in (("d", 0), ("d", 8193), ("n", -1), ("type", 3), ("stream_type", 1), ("kind", 2), ("gate_mode", 3), ("gate_mode", 1), ("gate_activation", 9), ("pre_norm", 0)):
        bad = HE.ResidualNorm(n=4, d=8, pre_norm=1, residual_scale=1.0)
        setattr(bad, field, value)
        assert L.marius_residual_norm_forward(C.byref(bad), P(x), 8, None, 0, None, 0, P(x), 8, None) == 1, field
    g = HE.ResidualNormGrads(grad_h=P(x), grad_h_ld=8, dx=P(x), dx_ld=8, dpre_weight=P(x))
    assert L.marius_residual_norm_backward(C.byref(m), C.byref(g), P(x), 8, None, 0, None, 0, None) == 1       # no workspace for the sum
    assert L.marius_residual_norm_backward(C.byref(m), None, P(x), 8, None, 0, None, 0, None) == 1


def test_neighbor_plan_refuses(HE):
    i64 = lambda *v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    f = HE.NeighborPlan
    refused(HE, "outside the 3 rows", f, i64(0, 3), i64(0), 3)
    refused(HE, "outside the 3 rows", f, i64(0, -1), i64(0), 3)
    refused(HE, "ascend", f, i64(0, 1), i64(1, 2), 3)
    refused(HE, "ascend", f, i64(0, 1, 2), i64(0, 2, 1), 3)
    refused(HE, "ascend", f, i64(0, 1, 2), i64(0, 4), 3)
    refused(HE, "ascend", f, i64(0, 1, 2), i64(0, -1), 3)
    refused(HE, "without a target", f, i64(0, 1), i64(), 3)
    refused(HE, "own row", f, i64(0, 1), i64(0, 1), 3, self_offset=2)
    refused(HE, "own row", f, i64(0, 1), i64(0, 1), 3, self_offset=-1)
    refused(HE, "int64", f, i64(0, 1).int(), i64(0), 3)
    refused(HE, "number of targets", f, i64(0), i64(0), 3, i64(0), i64(0, 1))
    refused(HE, "both", f, i64(0), i64(0), 3, i64(0))
    empty = f(i64(), i64(), 0)
    assert empty.num_entries == 0
    out, stats = HE.neighbor_attention(torch.zeros(0, 2, 4), torch.zeros(0, 2, 4), torch.zeros(0, 2, 4), empty)
    assert out.shape == (0, 2, 4) and stats.shape == (0, 2, 2)


def test_neighbor_attention_refuses(HE):
    plan = HE.NeighborPlan(torch.tensor([0, 1, 2]), torch.tensor([0, 1]), 3)
    q, k = torch.zeros(2, 4, 8), torch.zeros(3, 2, 8)
    f = HE.neighbor_attention
    refused(HE, "NeighborPlan is needed", f, q, k, k, None)
    refused(HE, "2 targets over 3 rows", f, q[:1], k, k, plan)
    refused(HE, "2 targets over 3 rows", f, q, k[:2], k[:2], plan)
    refused(HE, "multiple of the key heads", f, q[:, :3], k, k, plan)
    refused(HE, "required", f, q, k, k[:, :1], plan)
    refused(HE, "of one type", f, q, k.half(), k, plan)
    refused(HE, "1 to 256", f, torch.zeros(2, 1, 257), torch.zeros(3, 1, 257), torch.zeros(3, 1, 257), plan)
    refused(HE, "1 to 256", f, q, k[..., :4], k[..., :4], plan)
    refused(HE, "float32, bfloat16 or float16", f, q.double(), k.double(), k.double(), plan)
    refused(HE, "bias is float32", f, q, k, k, plan, None, torch.zeros(3, 3))
    refused(HE, "bias is float32", f, q, k, k, plan, None, torch.zeros(3, 4).half())
    _, stats = f(q, k, k, plan)
    b = HE.neighbor_attention_backward
    refused(HE, "not like the output", b, q[:1], q, k, k, stats, plan)
    refused(HE, "not like the output", b, q.half(), q, k, k, stats, plan)
    refused(HE, "stats is float32", b, q, q, k, k, stats[:1], plan)


def test_adamw_refuses(HE):
    p, s = [torch.zeros(300)], [torch.zeros(300)]
    f8, sc = [torch.zeros(300).to(torch.float8_e4m3fn)], [torch.zeros(2)]
    refused(HE, "no parameters", HE.AdamWTensors, [], [], [])
    refused(HE, "different lengths", HE.AdamWTensors, p, s, s + s)
    refused(HE, "different lengths", HE.AdamWTensors, p, f8, f8, sc)
    refused(HE, "contiguous", HE.AdamWTensors, [torch.zeros(300, 2)[:, 0]], s, s)
    refused(HE, "of its size", HE.AdamWTensors, p, [s[0].half()], s)
    refused(HE, "of its size", HE.AdamWTensors, p, [s[0][:5]], s)
    refused(HE, "one for 256", HE.AdamWTensors, p, f8, f8, sc, [torch.zeros(1)])
    refused(HE, "of its size", HE.AdamWTensors, p, s, s, sc, sc)
    t = HE.AdamWTensors(p, s, [torch.zeros(300)])
    refused(HE, "AdamWTensors are needed", HE.adamw_step, p, s, 1)
    refused(HE, "gradients for", HE.adamw_step, t, [], 1)
    refused(HE, "gradient 0 is not", HE.adamw_step, t, [torch.zeros(299)], 1)
    refused(HE, "float32, bfloat16 or float16 gradients", HE.adamw_step, t, [torch.zeros(300).double()], 1)
    refused(HE, "counted from 1", HE.adamw_step, t, s, 0)
    refused(HE, "betas in", HE.adamw_step, t, s, 1, beta1=1.0)
    refused(HE, "one int64", HE.adamw_step, t, s, torch.tensor([1.0]))
    refused(HE, "one float32", HE.adamw_step, t, s, 1, grad_scale=torch.zeros(2))
    refused(HE, "not a dense tensor", HE.adamw_step, t, [torch.zeros(300).to_sparse()], 1)
    refused(HE, "twice", HE.AdamWTensors, p + p, s + [torch.zeros(300)], [torch.zeros(300), torch.zeros(300)])
    flat = torch.zeros(500)
    refused(HE, "overlaps", HE.AdamWTensors, [flat[:300], flat[200:]], s + [torch.zeros(300)], [torch.zeros(300), torch.zeros(300)])
    refused(HE, "twice", HE.AdamWTensors, p, s, s)
    p[0].data = torch.zeros(301)
    refused(HE, "no longer", HE.adamw_step, t, s, 1)


# ------------------------------------------------------------------------------------------------ the reference itself
@pytest.mark.parametrize("kind", ["RMS", "LAYER"])
def test_reference_norm_gradients_are_autograds(kind):
    torch.manual_seed(0)
    x, z, gy, gh = (torch.randn(5, 7, dtype=torch.float64) for _ in range(4))
    y = x.clone().requires_grad_(True)
    yn, r, m = R.norm_rows(y, kind, 1e-3)
    yn.backward(gh)
    d, _ = R.norm_back(gh, gh.abs(), yn.detach(), m.detach(), r.detach(), kind)
    assert torch.allclose(d, y.grad, rtol=1e-12, atol=1e-13)
    want = torch.nn.functional.layer_norm(x, (7,), eps=1e-3) if kind == "LAYER" else torch.nn.functional.rms_norm(x, (7,), eps=1e-3)
    assert torch.allclose(R.norm_rows(x, kind, 1e-3)[0], want, rtol=1e-12)


def test_reference_attention_gradients_are_autograds():
    index, offsets = T.lists(4, 6, [3, 0, 5, 1], 0)
    rows, owner = R.lists_of(index, offsets, 4)
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, bias, grad = rnd(4, 4, 5), rnd(6, 2, 5), rnd(6, 2, 5), rnd(9, 4), rnd(4, 4, 5)
    bias[2] = -math.inf
    got = R.attention(q, k, v, rows, owner, 0.5, bias, grad)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, bias)]
    out = torch.zeros(4, 4, 5, dtype=torch.float64)
    for i in range(4):
        at = (owner == i).nonzero().flatten()
        for h in range(4):
            if at.numel():
                p = torch.softmax(leaves[1][rows[at], h // 2] @ leaves[0][i, h] * 0.5 + leaves[3][at, h], 0)
                out = out.index_put((torch.tensor(i), torch.tensor(h)), p @ leaves[2][rows[at], h // 2])
    assert torch.allclose(out, got["out"][0], rtol=1e-12, atol=1e-13)
    out.backward(grad)
    for name, leaf in zip(("dq", "dk", "dv", "dbias"), leaves):
        assert torch.allclose(got[name][0], leaf.grad, rtol=1e-10, atol=1e-12), name


def test_emulated_encoder_and_optimizer(HE):
    from marius_amd import gnn

    for bits, inc, out in ((32, True, True), (8, True, False)):
        T.test_attention_encoder_steps(HE, gnn, CPU, bits, inc, out)
    T.test_attention_plan_places_of_two_lists(HE, CPU)
    T.test_optimizer_state_is_saved_and_loaded(HE, CPU)


def test_emulated_small_forms(HE):
    from marius_amd import gnn

    T.test_residual_norm_of_tiny_rows_without_eps(HE, CPU)
    T.test_second_derivatives_are_refused(HE, gnn, CPU)
    T.test_gradient_of_a_sum_reaches_every_operand(HE, gnn, CPU)


def test_encoder_modules_refuse(HE):
    from marius_amd import gnn
    from marius_amd.optim import AdamW

    graph = T.sampled(gnn, CPU, 50, 300, [4], True, True, 5, 1)
    graph.performMap()
    assert int(graph.entryRelations(5).max()) == 5
    refused(HE, "outside the 3 relations", graph.entryRelations, 3)
    pairs = T.sampled(gnn, CPU, 50, 300, [4], True, False, 5, 1)
    pairs.performMap()
    pairs.dst_sorted_edges_ = pairs.dst_sorted_edges_[:, [0, 2]].contiguous()
    refused(HE, "three columns", pairs.entryRelations, 5)

    refused(HE, "multiple of the number of heads", gnn.GraphAttentionLayer, 8, 10, 4, device=CPU)
    refused(HE, "comes with the call", gnn.ResidualNorm(4, gate="ELEMENT", device=CPU), torch.zeros(2, 4), torch.zeros(2, 4))
    refused(HE, "comes with the call", gnn.ResidualNorm(4, device=CPU), torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(2, 4))
    refused(HE, "no parameters", AdamW, [])
    refused(HE, "32 or in 8", AdamW, [torch.zeros(3)], state_bits=16)


def test_emulated_single_rows_nan_gates_and_absent_gradients(HE):
    from marius_amd import gnn

    T.test_views_of_one_row_may_have_any_stride(HE, CPU)
    for gate in ("channel", "element"):
        T.test_nan_goes_through_a_relu_gate(HE, CPU, gate)
    T.test_norm_without_a_gradient_of_its_stream(HE, gnn, CPU)
    T.test_adamw_step_is_seen_by_graphs_that_saved_the_parameter(HE, CPU)
    T.test_a_refused_optimizer_step_does_not_count(HE, CPU)


@pytest.mark.parametrize("entries,heads,bins", [(0, 3, 5), (9, 4, 6), (777, 5, 256), (300, 100, 3), (2049, 33, 41)])
def test_emulated_bin_sum(HE, entries, heads, bins):
    T.test_bin_sum(HE, CPU, entries, heads, bins)


def test_emulated_layer_with_many_relations(HE):
    from marius_amd import gnn

    T.test_attention_layer_with_more_relations_than_bins(HE, gnn, CPU)
    T.test_attention_layer_in_bfloat16(HE, gnn, CPU)


def test_bin_sum_refuses(HE):
    v, b = torch.zeros(4, 3), torch.zeros(4, dtype=torch.int64)
    refused(HE, "float32 \\[entries, heads\\]", HE.bin_sum, v.double(), b, 2)
    refused(HE, "float32 \\[entries, heads\\]", HE.bin_sum, v[0], b, 2)
    refused(HE, "float32 \\[entries, heads\\]", HE.bin_sum, torch.zeros(4, 0), b, 2)
    refused(HE, "int64 bin for every", HE.bin_sum, v, b.int(), 2)
    refused(HE, "int64 bin for every", HE.bin_sum, v, b[:3], 2)
    refused(HE, "1 to 256 bins", HE.bin_sum, v, b, 0)
    refused(HE, "1 to 256 bins", HE.bin_sum, v, b, 257)


def test_encoder_block_under_address_and_undefined_behaviour_sanitizers():
    """the forms above that reach every kernel at odd sizes, and every refusal, once more in a python started under libasan with the kernel files built with
    -fsanitize=address,undefined (libstdc++ is loaded with it: the host module's refusals are C++ exceptions)"""
    if os.environ.get("MARIUS_EMUL_SANITIZE") == "1":
        pytest.skip("already inside the sanitizer run")
    libraries = [subprocess.run(["gcc", "-print-file-name=" + name], stdout=subprocess.PIPE, text=True).stdout.strip() for name in ("libasan.so", "libstdc++.so")]
    if not all(os.path.isabs(p) and os.path.exists(p) for p in libraries):
        pytest.skip("no libasan.so next to gcc")
    env = dict(os.environ, MARIUS_EMUL_SANITIZE="1", LD_PRELOAD=" ".join(libraries), ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    select = "not sanitizers" if os.environ.get("MARIUS_EMUL_SANITIZE_ALL") == "1" else "small_forms or single_rows or refuse or adamw or bin_sum or masks or (residual_norm and 2047) or (single and 256)"
    r = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-x", "-q", "-p", "no:cacheprovider", "-k", select], env=env, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=2400, cwd=os.path.dirname(HERE))
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-4000:]
