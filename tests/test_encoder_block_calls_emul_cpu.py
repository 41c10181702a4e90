"""tests/test_gpu_encoder_block_calls.py on the CPU build of its kernel files (tests/emul), and what is refused there."""
import ctypes as C
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

import test_gpu_encoder_block_calls as T  # noqa: E402
from test_encoder_block_emul_cpu import CPU, refused  # noqa: E402
from test_kernels_emul_cpu import HE, emulated_library  # noqa: E402,F401  (fixtures)

F32, BF16, F16 = T.F32, T.BF16, T.F16


@pytest.mark.parametrize("masked", [None, 2, 6])
def test_emulated_log_sum_exp(HE, masked):
    T.test_log_sum_exp_beside_the_output(HE, CPU, masked, 8, 2, 64, BF16)
    T.test_log_sum_exp_beside_the_output(HE, CPU, masked, 4, 4, 25, F32)


# ------------------------------------------------------------------------------------------------ refusals
def test_residual_norm_refuses_wide_rows_even_where_there_are_none(HE):
    """gradients of weights over 8192 elements, which nothing would have written"""
    x, w = torch.zeros(0, 9000), torch.ones(9000)
    refused(HE, "1 to 8192", HE.residual_norm, x, pre_weight=w)
    refused(HE, "1 to 8192", HE.residual_norm_backward, x, x, x, x, w, w, w, w, w, post_norm=True)
    got = HE.residual_norm_backward(*(torch.zeros(0, 8192) for _ in range(4)), *(torch.ones(8192) for _ in range(5)), post_norm=True)
    assert all(not got[k].any() for k in ("dgate", "dpost_weight", "dpost_bias", "dpre_weight", "dpre_bias"))
    assert HE.residual_norm(torch.zeros(0, 0))[1].shape == (0, 0)


def test_neighbor_attention_c_abi_refuses_plans_without_their_arrays(HE):
    """the kernels read numbers of every work item, an empty list's too, and a list is written by its item: what a plan says that it has has to be there"""
    L, P = HE.lib(), HE.ptr
    q, k, out, stats, ws = torch.ones(2, 1, 4), torch.ones(3, 1, 4), torch.zeros(2, 1, 4), torch.zeros(2, 1, 2), torch.zeros(4096)
    dk, dv, bias = torch.zeros(3, 1, 4), torch.zeros(3, 1, 4), torch.zeros(1)
    plan = HE.NeighborPlan(torch.zeros(0, dtype=torch.int64), torch.zeros(2, dtype=torch.int64), 3)
    assert plan.desc.n_items == 2 and plan.desc.r_n_items == 3 and plan.num_entries == 0

    def calls(**change):
        d = HE.NeighborPlanDesc.from_buffer_copy(plan.desc)
        for name, value in change.items():
            setattr(d, name, value)
        m = HE.NeighborAttention(heads=1, kv_heads=1, dim=4, scale=1.0, q=q.data_ptr(), k=k.data_ptr(), v=k.data_ptr(), q_row=4, k_row=4, v_row=4, stats=stats.data_ptr())
        forward = L.marius_neighbor_attention_forward(C.byref(d), C.byref(m), P(out), P(ws), 16384, None)
        m.bias = bias.data_ptr()
        return forward, L.marius_neighbor_attention_backward(C.byref(d), C.byref(m), P(q), 4, 4, P(out), P(dk), P(dv), None, P(ws), 16384, None)

    assert calls() == (0, 0)
    assert calls(index=None) == (1, 1) and calls(items=None) == (1, 1)
    assert calls(n_items=1) == (1, 1) and calls(n_splits=1, n_slots=2, splits=None) == (1, 1)      # fewer items than lists; a cut list without its parts
    for change in (dict(r_owner=None), dict(r_entry=None), dict(r_items=None), dict(r_n_items=2), dict(r_n_splits=1, r_n_slots=2, r_splits=None)):
        assert calls(**change) == (0, 1), change


# ------------------------------------------------------------------------------------------------ graphs and encoders
@pytest.fixture()
def G(HE):
    from marius_amd import gnn

    return gnn


def test_emulated_plans_are_of_mapped_lists(HE, G):
    T.test_plans_are_of_mapped_lists(HE, G, CPU)


@pytest.mark.parametrize("out_edges", [[[2, 1, 3]], []])
@pytest.mark.parametrize("in_edges", [[[3, 0, 2], [2, 4, 1], [1, 2, 0]], [[3, 3, 2]], []])
def test_emulated_encoder_over_layers_whose_lists_run_out(HE, G, in_edges, out_edges):
    T.test_encoder_over_layers_whose_lists_run_out(HE, G, CPU, in_edges, out_edges)


# ------------------------------------------------------------------------------------------------ AdamW
@pytest.mark.parametrize("capturable", [False, True])
def test_emulated_refused_steps(HE, capturable):
    for what in range(4):
        T.test_a_refused_step_changes_nothing(HE, CPU, what, capturable)


@pytest.mark.parametrize("bits", [32, 8])
def test_emulated_gradients_that_are_not_contiguous(HE, bits):
    T.test_gradients_that_are_not_contiguous(HE, CPU, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_emulated_gradients_that_are_not_finite(HE, bits):
    T.test_gradients_that_are_not_finite_spoil_no_more_than_they_have_to(HE, CPU, bits)


def test_adamw_check_refuses_and_does_nothing(HE):
    p, m, v = (torch.ones(300) for _ in range(3))
    t = HE.AdamWTensors([p], [m], [v])
    refused(HE, "gradient 0 is not", HE.adamw_check, t, [torch.zeros(299)], 1)
    refused(HE, "counted from 1", HE.adamw_check, t, [p], 0)
    refused(HE, "AdamWTensors are needed", HE.adamw_check, [p], [p], 1)
    HE.adamw_check(t, [torch.ones(300)], 1)
    assert all(bool((x == 1).all()) for x in (p, m, v))
    L, table = HE.lib(), HE.AdamWTensor(param=p.data_ptr(), grad=p.data_ptr(), exp_avg=m.data_ptr(), exp_avg_sq=v.data_ptr(), n=300)
    call = lambda table, *a: L.marius_adamw_check(table, 1, 0, 0, 32, *a)  # noqa: E731
    assert call(C.byref(table), 1, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0) == 0
    for bad in ((0, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0), (1, None, 1, float("nan"), 0.9, 0.999, 1e-8, 0.0), (1, None, 1, 1e-3, 1.0, 0.999, 1e-8, 0.0), (1, None, 1, 1e-3, 0.9, 0.999, -1.0, 0.0),
                (0, p.data_ptr(), 2, 1e-3, 0.9, 0.999, 1e-8, 0.0)):
        assert call(C.byref(table), *bad) == 1, bad
    assert call(None, 1, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0) == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_emulated_counts_of_steps(HE, bits):
    for capturable in (False, True):
        T.test_every_parameter_counts_its_own_steps(HE, CPU, bits, capturable)


def test_emulated_steps_on_the_device(HE):
    for count in (3, 70):
        T.test_a_step_on_the_device_for_every_tensor(HE, CPU, count)
    T.test_steps_of_tensors_far_apart_in_a_long_list(HE, CPU)


# ------------------------------------------------------------------------------------------------ residual norm
def test_emulated_sigmoid_gates_far_from_zero(HE):
    for gate in ("channel", "element"):
        for kind in (F32, BF16):
            T.test_sigmoid_gates_far_from_zero(HE, CPU, gate, kind)


# ------------------------------------------------------------------------------------------------ plans
def test_emulated_plan_is_recorded_whole(HE):
    T.test_a_plan_in_use_on_another_stream_is_recorded_whole(HE, CPU)


def test_emulated_plan_keeps_no_hold_on_its_lists(HE):
    T.test_a_plan_keeps_no_hold_on_the_lists_it_was_made_of(HE, CPU)


def test_neighbor_plan_refuses_offsets_of_lists_that_are_not_there(HE):
    """offsets over an index of no entries are zeros: others belong to another index"""
    i64 = lambda *v: torch.tensor(v, dtype=torch.int64)  # noqa: E731
    for bad in (i64(0, 3), i64(1, 1), i64(0, -1)):
        refused(HE, "ascend", HE.NeighborPlan, i64(), bad, 3)
        refused(HE, "ascend", HE.NeighborPlan, i64(0, 1, 2), i64(0, 2), 3, i64(), bad)
        refused(HE, "ascend", HE.NeighborPlan, i64(), bad, 3, i64(0, 1, 2), i64(0, 2), self_offset=1)
    plan = HE.NeighborPlan(i64(), i64(0, 0), 3, i64(0, 1, 2), i64(0, 2), self_offset=1)
    assert plan.num_entries == 5 and plan.places(0).numel() == 0 and plan.places(1).tolist() == [0, 1, 3] and plan.places("own").tolist() == [2, 4]


def test_emulated_parameters_given_one_memory(HE):
    T.test_parameters_given_one_memory_after_their_optimizer_was_made(HE, CPU)


def test_emulated_states_given_new_memory(HE):
    T.test_states_given_new_memory(HE, CPU)


def test_residual_norm_module_refuses_gates_it_would_leave_out(HE, G):
    refused(HE, "gate is one of", G.ResidualNorm, 4, gate="channel", device=CPU)
    refused(HE, "gate is one of", G.GraphAttentionEncoder, 4, 8, 2, 1, 2, gate=None, device=CPU)
    for gate in ("NONE", "CHANNEL", "ELEMENT"):
        refused(HE, "without a block", G.ResidualNorm(4, gate=gate, device=CPU), torch.zeros(2, 4), None, torch.zeros(2, 4))


def test_adagrad_refuses_parameters_that_are_not_float32(HE, G):
    """an encoder in bfloat16 goes forward and back, but the Adagrad step reads and writes four bytes an element"""
    import test_gpu_encoder_block as B

    graph = B.sampled(G, CPU, 50, 400, [4], True, True, 6, 1)
    enc = G.GraphAttentionEncoder(6, 8, 3, 1, 4, device=CPU).bfloat16()
    x, labels = torch.randn(graph.node_ids_.numel(), 6).bfloat16(), torch.zeros(6, dtype=torch.int64)
    refused(HE, "float32", G.node_classification_step, enc, x, graph, labels, 0.1)
    assert all(p.grad is None for p in enc.parameters())                       # before the pass
    w, s = torch.ones(8), torch.ones(8)
    for bad in ((w.bfloat16(), s, w), (w, s.half(), w), (w, s, w.double()), (w, s[:4], w), (w, s, torch.ones(16)[::2]), (torch.ones(16)[::2], s, w)):
        refused(HE, "float32", HE.dense_adagrad_step, *bad, 0.1)
    HE.dense_adagrad_step(w, s, torch.ones(8), 0.1)
    assert bool((w < 1).all())
