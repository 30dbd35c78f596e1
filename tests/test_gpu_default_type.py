"""Bound queries on fp32 networks give the same bits whatever torch's default type is (a program whose own networks
are 16-bit sets it)."""

import pytest
import torch

from boundflow_amd import alpha_beta as hab
from boundflow_amd import bab as hbab
from boundflow_amd import crown as hc
from boundflow_amd import task_executor as te
from boundflow_amd import workloads as wl
from tests.gpu_util import announce, device

pytestmark = pytest.mark.gpu


def queries(dev):
    mlp = wl.to_device(wl.subset(wl.make_c1(), 8), dev)
    cnn = wl.to_device(wl.subset(wl.make_c3(), 3), dev)
    dag = wl.to_device(wl.make_dag("residual_mlp"), dev)
    conv_dag = wl.to_device(wl.make_dag("projection_skip_cnn"), dev)
    toy = wl.to_device(wl.make_bab_toy(batch=2), dev)
    ibp = wl.to_device(wl.make_ibp_dag(), dev)

    def pair(b):
        return [b.lower, b.upper]

    def crown(w):
        return lambda: pair(hc.run_crown_ibp_mlp(w.module, w.spec, linear_spec_C=w.C))

    def alpha(w):
        return lambda: pair(hab.run_alpha_crown_mlp(w.module, w.spec, linear_spec_C=w.C, steps=3, lr=0.2)[0])

    def tree():
        r = hbab.solve_bab_mlp(toy.module, toy.spec, linear_spec_C=toy.C,
                               config=hbab.BabConfig(max_nodes=20, oracle="alpha_beta", node_batch_size=8, alpha_steps=3))
        return [torch.tensor([[p.best_lower, p.best_upper, p.nodes_visited] for p in r.per_example],
                             dtype=torch.float64)]

    def intervals():
        out = te.HipTaskExecutor().run_ibp(ibp.module, ibp.spec)
        return pair(out)

    return {"mlp": crown(mlp), "cnn": crown(cnn), "dag": crown(dag), "conv dag": crown(conv_dag),
            "alpha mlp": alpha(mlp), "alpha cnn": alpha(cnn), "alpha dag": alpha(dag), "alpha conv dag": alpha(conv_dag),
            "tree": tree, "intervals": intervals}


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_bounds_do_not_depend_on_the_default_type(default):
    dev = device()
    # networks of its own for each side: nothing that a query keeps of a weight is there already
    for (name, query), other in zip(queries(dev).items(), queries(dev).values()):
        announce(f"{name} under {default}")
        want = other()
        before = torch.get_default_dtype()
        torch.set_default_dtype(default)
        try:
            got = query()
        finally:
            torch.set_default_dtype(before)
        for a, b in zip(got, want, strict=True):
            assert a.dtype == b.dtype and torch.equal(a, b), name
