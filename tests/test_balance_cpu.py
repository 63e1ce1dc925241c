"""What a layer counts for its balance belongs to its process: parallel training, casts, copies (CPU)."""
from __future__ import annotations

import copy
import datetime
import os
import pickle

import pytest
import torch
import torch.multiprocessing as mp

import fastmoe_amd as fm
from fastmoe_amd import moe as layers

E, K, D = 4, 2, 8


def make():
    torch.manual_seed(0)
    return fm.MoEFeedForward(D, 6, E, K, implementation=fm.MoEImplementation.STANDARD, routing=fm.Routing("sigmoid"),
                             balance=True)


def plain_gate_and_sort(x, router, top_k, num_experts, *, routing=None, bias=None):
    """The dispatch by torch's operators (the kernels take GPU tensors alone)."""
    B, T, width = x.shape
    flat = x.reshape(-1, width)
    s = torch.sigmoid(router(flat))
    ids = torch.topk(s + bias, top_k, dim=-1).indices
    order = torch.argsort(ids.view(-1), stable=True)
    token = order // top_k
    counts = torch.bincount(ids.view(-1), minlength=num_experts)
    return layers._Routed((flat[token], torch.tensor([len(token)]), counts.view(1, -1), token,
                           s.gather(1, ids).view(-1)[order], (B, T)), None)


def count(rank, store, out):
    os.environ["GLOO_SOCKET_IFNAME"] = "lo"  # the host's name need not resolve
    torch.distributed.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=2,
                                         timeout=datetime.timedelta(seconds=120))
    layers.gate_and_sort = plain_gate_and_sort  # in this process alone
    moe = make()
    ddp = torch.nn.parallel.DistributedDataParallel(moe, find_unused_parameters=True)  # an expert may have no rows
    want = torch.zeros(E, dtype=torch.int64)
    for step in range(3):  # several forwards before the balance is moved, other rows on each rank
        x = torch.randn(1, 5 + 4 * rank + step, D, generator=torch.Generator().manual_seed(10 * rank + step))
        want += plain_gate_and_sort(x, moe.router, K, E, bias=moe.balance_bias)[2].view(-1)
        ddp(x).sum().backward()
    mine = moe.expert_load.clone()
    torch.distributed.all_reduce(moe.expert_load)
    both = moe.expert_load.clone()
    moe.update_balance(0.25)
    torch.save((mine, want, both, moe.balance_bias), f"{out}{rank}")
    torch.distributed.destroy_process_group()


def test_each_process_keeps_its_own_counts(tmp_path):
    mp.spawn(count, (str(tmp_path / "store"), str(tmp_path / "out")), nprocs=2)
    a, b = (torch.load(tmp_path / f"out{r}") for r in range(2))
    assert torch.equal(a[0], a[1]) and torch.equal(b[0], b[1])
    assert int(a[0].sum()) == K * (5 + 6 + 7) and int(b[0].sum()) == K * (9 + 10 + 11)
    assert torch.equal(a[2], a[0] + b[0]) and torch.equal(b[2], a[2])
    assert torch.equal(a[3], b[3]) and bool(a[3].any())


def test_counts_are_no_state_and_stay_whole_numbers():
    moe = make()
    assert set(dict(moe.named_buffers())) == {"balance_bias"} and "expert_load" not in moe.state_dict()
    moe.expert_load += torch.arange(E)
    for cast in (lambda m: m.half(), lambda m: m.type(torch.float64), lambda m: m.to(torch.bfloat16), copy.deepcopy,
                 lambda m: pickle.loads(pickle.dumps(m))):
        got = cast(copy.deepcopy(moe))
        assert got.expert_load.dtype == torch.int64 and got.expert_load.tolist() == list(range(E))
        assert got.balance_bias.dtype == torch.float32
    other = copy.deepcopy(moe)
    other.expert_load.zero_()
    assert moe.expert_load.tolist() == list(range(E))
    bare = copy.deepcopy(moe).to("meta").to_empty(device="cpu")
    assert bare.expert_load.device.type == "cpu" and not bare.expert_load.any()
    assert fm.MoEFeedForward(D, 6, E, K).expert_load is None


@pytest.mark.parametrize("balance", [False, True])
def test_layers_pickled_with_their_counts_as_a_buffer(balance):
    moe = make() if balance else fm.MoEFeedForward(D, 6, E, K)
    state = copy.deepcopy(moe.__dict__)
    state.pop("expert_load")
    state["_buffers"]["expert_load"] = torch.arange(E) if balance else None
    state["_non_persistent_buffers_set"] = {"expert_load"}
    old = fm.MoEFeedForward.__new__(fm.MoEFeedForward)
    old.__setstate__(state)
    assert old.state_dict().keys() == moe.state_dict().keys()
    assert set(dict(old.named_buffers())) == ({"balance_bias"} if balance else set())
    assert old.expert_load.tolist() == list(range(E)) if balance else old.expert_load is None
