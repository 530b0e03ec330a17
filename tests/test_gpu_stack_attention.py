"""The layer stack with attention over the 4-bit cache: every stage of a layer against its plain form on the stage's own
inputs, through prefill, decode, a padded step and a captured one."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from velox_inferer_b200.stack import LinearStack, StackAttention, StackSpec

from . import kv4_ref as R
from .gpu_util import backend
from .test_gpu_kv4 import check, close_rows, f64, i32

pytestmark = pytest.mark.gpu
SPEC = StackSpec(layers=2, hidden=256, intermediate=512, heads=4, kv_heads=1, head_dim=128)


def check_last_layer(b, stack, att, new, lens, m):
    """The last layer's buffers still hold its step."""
    n, D = int(sum(new)), SPEC.head_dim
    st, c = att.step, att.caches[-1]
    assert st.status.item() == 0
    pos = np.concatenate([lens[i] + np.arange(new[i]) for i in range(len(new))])
    assert np.array_equal(st.positions.cpu().numpy()[:n], pos) and np.all(st.positions.cpu().numpy()[n:] == -1)
    q, k, v = (x[: m * h * D].view(m, h, D)[:n] for x, h in ((stack.qb, 4), (stack.kb, 1), (stack.vb, 1)))
    rope, ones = att.rope.cpu().numpy(), np.ones(D, np.float32)
    close_rows(att.qn[:n], f64(q), ones, SPEC.norm_eps, False, rope, pos, False)
    kk = R.norm_rope(f64(k), ones, SPEC.norm_eps, False, rope, pos, False).astype(np.float32)
    cache = R.Cache(c.storage.cpu().numpy(), att.page_size, D, c.k_divisor, c.v_divisor)
    want = R.Cache(np.zeros_like(cache.s), att.page_size, D, c.k_divisor, c.v_divisor)
    for t, slot in enumerate(st.slots.cpu().numpy()[:n]):
        want.write(int(slot), kk[t], f64(v)[t].astype(np.float32))
        for got, ref in zip(cache.read(int(slot)), want.read(int(slot))):
            assert np.array_equal(got, ref)
    cu = np.concatenate([[0], np.cumsum(new)])
    check(c, att.table.cpu().numpy(), cu, lens + new, att.qn[:n], att.out[:n], 0, D ** -0.5, True, 0)
    # the o projection reads the attention's result
    o = stack.layers[-1].o
    act = b.linear_act(o, m)
    x = att.out.float().cpu().numpy().reshape(m, -1)
    pb = torch.empty(m * SPEC.hidden, dtype=torch.bfloat16, device=b.device)
    b.linear_bf16(att.out, o, None, m, yb=pb)
    wanted = O.linear(x, o.buf.cpu().numpy(), O.FMT_NVFP4, o.parent_rows, o.k, 0, o.parent_rows, m,
                      act=O.ACT_NVFP4 if act.divisor else O.ACT_BF16, divisor=act.divisor)
    # the library's bound for an f32 result (1e-2 of the rms), and the rounding of this one to bf16 (2^-8 of the value)
    got = pb.float().cpu().numpy().reshape(m, -1)[:n]
    assert np.all(np.abs(got - wanted[:n]) <= 1e-2 * O.rms(wanted[:n]) + 2.0 ** -8 * np.abs(wanted[:n]))


def test_stack_with_attention():
    b = backend()
    requests, pages = 3, 30
    stack = LinearStack(b, SPEC, max_tokens=80, a4=True, seed=5)
    g = torch.Generator(device=b.device).manual_seed(0)
    lens = np.zeros(requests, np.int64)
    atts = {}

    def step(new, m, shared):
        """A step of m rows; the caches, pages and lengths carry on from the step before."""
        att = StackAttention(b, SPEC, requests, m, pages, page_size=16, max_positions=400)
        if shared is not None:
            att.caches, att.table, att.taken, att.cached = shared.caches, shared.table, shared.taken, shared.cached
        xb = torch.randn(m, SPEC.hidden, generator=g, device=b.device).to(torch.bfloat16)
        att.plan(i32(new), max(new))
        out = stack.forward(xb, m, att)
        assert torch.isfinite(out[: int(sum(new)) * SPEC.hidden]).all()
        check_last_layer(b, stack, att, np.array(new), lens, m)
        return att

    att = None
    for new, m in (([40, 1, 30], 71), ([1, 17, 1], 24), ([1, 1, 1], 3), ([0, 5, 1], 6)):
        att = step(new, m, att)
        lens = lens + np.array(new)
    # a captured decode step, replayed while the lengths grow
    dec = StackAttention(b, SPEC, requests, 3, pages, page_size=16, max_positions=400)
    dec.caches, dec.table, dec.taken, dec.cached = att.caches, att.table, att.taken, att.cached
    one, xb = i32([1, 1, 1]), torch.zeros(3, SPEC.hidden, dtype=torch.bfloat16, device=b.device)

    def decode():
        dec.plan(one, 1)
        return stack.forward(xb, 3, dec)

    decode()                                              # eager once, before the capture
    lens = lens + 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode()
    for i in range(20):
        xb.copy_(torch.randn(3, SPEC.hidden, generator=g, device=b.device))
        graph.replay()
        torch.cuda.synchronize()
        if i in (0, 7, 19):
            check_last_layer(b, stack, dec, np.array([1, 1, 1]), lens, 3)
        lens = lens + 1
    assert b.debug_status() == 0


def test_stack_without_attention_is_unchanged():
    """The passthrough step gives the same bits whether or not an attention was made for the stack."""
    b = backend()
    stack = LinearStack(b, SPEC, max_tokens=40, a4=True, seed=5)
    xb = torch.randn(40, SPEC.hidden, generator=torch.Generator(device=b.device).manual_seed(1), device=b.device).to(torch.bfloat16)
    first = stack.forward(xb, 40).clone()
    att = StackAttention(b, SPEC, 1, 40, 9, page_size=16, max_positions=64)
    att.plan(i32([40]))
    other = stack.forward(xb, 40, att).clone()
    assert torch.equal(stack.forward(xb, 40), first) and not torch.equal(other, first)
