"""Tensors that the drafting operators refuse for where they lie, with an error and nothing launched."""
import pytest
import torch

from test_attention_few_gpu import make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tileinfer_b200.kernels import ops
    return ops


def attention_args(nq=4, nkv=2, dim=64):
    d = {key: t.cuda() for key, t in make([(2, 70)], nq, nkv, dim).items()}
    return dict(out=torch.zeros(2, nq * dim, dtype=torch.bfloat16, device="cuda"), q=d["q"], k_cache=d["k"], v_cache=d["v"], block_table=d["table"],
                seq_slots=d["seq_slots"], cu_seqlens=d["cu"], kv_lens=d["lens"], scale=0.1, nq=nq, nkv=nkv, head_dim=dim, page_size=64, max_new=2)


def shifted(t, by):
    """The same values in a contiguous view that begins ``by`` elements further on."""
    held = torch.zeros(t.numel() + by, dtype=t.dtype, device="cuda")
    held[by:].copy_(t.reshape(-1))
    return held[by:].view(t.shape)


def test_attention_queries_and_outputs_at_odd_places(ops):
    args = attention_args()
    ops.attention_few(**args)
    want = args["out"].clone()
    for name in ("q", "out"):
        with pytest.raises(ops.KernelError, match="4-byte aligned"):
            ops.attention_few(**{**args, name: shifted(args[name], 1)})
    out = shifted(torch.zeros_like(want), 2)
    ops.attention_few(**{**args, "q": shifted(args["q"], 2), "out": out})
    assert torch.equal(out, want)


def linear_args(n=20, out=1024, k=4096):
    codes = torch.zeros(out, k // 8, dtype=torch.int32, device="cuda")
    return dict(y=torch.zeros(n, out, dtype=torch.bfloat16, device="cuda"), x=torch.ones(n, k, dtype=torch.bfloat16, device="cuda"), codes=codes,
                scales=torch.ones(k // 128, out, dtype=torch.bfloat16, device="cuda"))


def test_linear4_work_spaces(ops):
    args, need = linear_args(), ops.linear4_workspace(20, 1024, 4096)
    held = torch.empty(2 * need, dtype=torch.uint8, device="cuda")
    ops.linear4(**args, workspace=held[:need])
    want = args["y"].clone()
    ops.linear4(**args, workspace=held[16:])
    assert torch.equal(args["y"], want)
    for ws in (held[1:], held[4:], held[:need - 1], held.cpu()):
        with pytest.raises(ops.KernelError, match="work space"):
            ops.linear4(**args, workspace=ws)


@pytest.mark.parametrize("what", ["attention_few", "linear4"])
def test_work_spaces_that_are_none(ops, what):
    """On the host, of another type, with holes, or one byte seen many times: refused before anything is launched."""
    args = attention_args() if what == "attention_few" else linear_args()
    need = ops.attention_few_workspace(1, 2, 4, 2, 64) if what == "attention_few" else ops.linear4_workspace(20, 1024, 4096)
    held = torch.empty(2 * need, dtype=torch.uint8, device="cuda")
    getattr(ops, what)(**args, workspace=held)
    for ws in (held.cpu(), held[:1].expand(2 * need), held[::2], held[:need // 4 * 4].view(torch.int32), held[:need - 1], held[8:]):
        with pytest.raises(ops.KernelError, match="work space"):
            getattr(ops, what)(**args, workspace=ws)


def test_attention_caches_of_other_dimensions(ops):
    """A cache is [pages, heads, 64, head size]: with one dimension more, its first is not the number of pages (those beyond it read as zeros)."""
    args = attention_args()
    k, v = args["k_cache"], args["v_cache"]
    pages = k.shape[0]
    for change in ((k[None], v[None]), (k.view(1, pages, 1, 2, 64, 64), v.view(1, pages, 1, 2, 64, 64)), (k[0], v[0])):
        with pytest.raises(ops.KernelError, match="do not fit"):
            ops.attention_few(**{**args, "k_cache": change[0], "v_cache": change[1]})
