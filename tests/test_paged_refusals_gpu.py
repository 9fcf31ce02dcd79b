"""What the paged operators refuse of tensors on the device -- before anything is launched: the outputs stay as they were."""
import pytest
import torch

from sequoia_amd import native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, KV, D, PAGE, ROWS, SEQS = 4, 2, 64, 16, 5, 2


@pytest.fixture(scope="module")
def ops():
    from sequoia_amd.ops import HipOps
    return HipOps()


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16, device=DEV)


def ints(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def pages():
    return dict(k_pages=half(3, KV, PAGE, D), v_pages=half(3, KV, PAGE, D), page_table=ints(0, 1, 2, 0).view(SEQS, 2))


def write_args():
    return dict(pages(), qkv=half(ROWS, (H + 2 * KV) * D), q_out=half(H, ROWS, D), cos=half(8, D), sin=half(8, D),
                position_ids=torch.arange(ROWS, device=DEV), seq_lens=ints(0, 1), cu_rows=ints(0, 2, ROWS), n_heads=H, h_kv=KV, d=D)


def read_args():
    return dict(pages(), k_out=half(SEQS, KV, 8, D), v_out=half(SEQS, KV, 8, D), starts=ints(0, 0), counts=ints(4, 4))


def attend_args():
    return dict(pages(), q=half(H, ROWS, D), out=half(ROWS, H * D), seq_lens=ints(0, 1), cu_rows=ints(0, 2, ROWS), scale=0.125)


def verify_args():
    return dict(target_logits=half(5, 40), draft_logits=half(3, 40), draft_tokens=ints(1, 2, 3, dtype=torch.int64), cu_drafts=ints(0, 1, 3),
                u_accept=torch.zeros(3, device=DEV), u_next=torch.zeros(2, device=DEV), temperature=1.0, n_accepted=ints(-7, -7),
                next_tokens=ints(-7, -7, dtype=torch.int64))


CALLS = {"rope_kv_write_paged": (write_args, ("q_out", "k_pages", "v_pages")), "kv_read_paged": (read_args, ("k_out", "v_out")),
         "paged_attention": (attend_args, ("out",)), "verify_drafts": (verify_args, ("n_accepted", "next_tokens"))}
TENSORS = [(call, name) for call, (make, _) in CALLS.items() for name in
           {"rope_kv_write_paged": ("qkv", "q_out", "k_pages", "v_pages", "cos", "sin", "position_ids", "page_table", "seq_lens", "cu_rows"),
            "kv_read_paged": ("k_pages", "v_pages", "k_out", "v_out", "page_table", "starts", "counts"),
            "paged_attention": ("q", "k_pages", "v_pages", "out", "page_table", "seq_lens", "cu_rows"),
            "verify_drafts": ("target_logits", "draft_logits", "draft_tokens", "cu_drafts", "u_accept", "u_next", "n_accepted", "next_tokens")}[call]]


def refused(ops, call, error, **changes):
    make, outputs = CALLS[call]
    args = make()
    args.update(changes)
    before = [args[o].clone() if isinstance(args[o], torch.Tensor) else None for o in outputs]
    with pytest.raises(error):
        getattr(ops, call)(**args)
    torch.cuda.synchronize()
    for o, b in zip(outputs, before):
        assert b is None or torch.equal(args[o], b)


@pytest.mark.parametrize("call", CALLS)
def test_the_calls_that_the_changes_below_start_from_are_taken(ops, call):
    make, outputs = CALLS[call]
    args = make()
    got = getattr(ops, call)(**args)
    torch.cuda.synchronize()
    if call in ("kv_read_paged", "verify_drafts"):
        assert got[0] is args[outputs[0]] and got[1] is args[outputs[1]]
    if call == "paged_attention":
        assert got is args["out"]


@pytest.mark.parametrize("call,name", TENSORS)
def test_wrong_types_places_and_things(ops, call, name):
    t = CALLS[call][0]()[name]
    refused(ops, call, TypeError, **{name: t.to(torch.float64)})
    refused(ops, call, TypeError, **{name: None})
    refused(ops, call, TypeError, **{name: 5})
    refused(ops, call, (ValueError, native.SequoiaNativeError), **{name: t.cpu()})


@pytest.mark.parametrize("call,name", TENSORS)
def test_wrong_shapes(ops, call, name):
    t = CALLS[call][0]()[name]
    refused(ops, call, ValueError, **{name: t[None].contiguous()})
    if name not in ("page_table", "cos", "sin", "k_pages", "v_pages", "n_accepted", "draft_tokens"):      # (their own sizes count)
        refused(ops, call, ValueError, **{name: t[:-1].contiguous()})
    if t.dim() > 1:
        refused(ops, call, ValueError, **{name: t[..., :-1]})
        refused(ops, call, ValueError, **{name: torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype, device=DEV)[..., ::2]})
    elif t.shape[0] > 1:
        refused(ops, call, ValueError, **{name: torch.zeros(2 * t.shape[0], dtype=t.dtype, device=DEV)[::2]})


def codes():
    return torch.zeros((3, KV, PAGE, D), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)


@pytest.mark.parametrize("call", ["rope_kv_write_paged", "kv_read_paged", "paged_attention"])
def test_scales_and_the_types_of_pages(ops, call):
    s = torch.full((3, KV, PAGE), 127, dtype=torch.uint8, device=DEV)
    refused(ops, call, ValueError, k_pages=codes(), v_pages=codes(), k_scales=s)
    refused(ops, call, ValueError, k_pages=codes(), v_pages=codes(), v_scales=s)
    refused(ops, call, TypeError, k_pages=codes(), v_pages=codes())
    refused(ops, call, TypeError, k_scales=s, v_scales=s)
    refused(ops, call, TypeError, k_pages=codes(), v_pages=codes(), k_scales=s, v_scales=s.int())
    refused(ops, call, ValueError, k_pages=codes(), v_pages=codes(), k_scales=s, v_scales=s[:, :, :8].contiguous())
    refused(ops, call, ValueError, k_pages=codes(), v_pages=codes(), k_scales=s, v_scales=s.transpose(0, 2).contiguous().transpose(0, 2))
    refused(ops, call, native.SequoiaNativeError, **{n: half(3, KV, 24, D) for n in ("k_pages", "v_pages")})       # no page size of the kernels'


def test_numbers(ops):
    refused(ops, "rope_kv_write_paged", ValueError, n_heads=3)
    refused(ops, "rope_kv_write_paged", ValueError, h_kv=1)
    refused(ops, "rope_kv_write_paged", ValueError, d=128)
    refused(ops, "rope_kv_write_paged", ValueError, n_heads=1 << 40)
    refused(ops, "rope_kv_write_paged", TypeError, n_heads=4.0)
    for bad in (-1, 9):
        refused(ops, "kv_read_paged", ValueError, max_count=bad)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused(ops, "paged_attention", ValueError, scale=bad)
    refused(ops, "paged_attention", native.SequoiaNativeError, scale=1e300)                                       # no fp32 number
    refused(ops, "paged_attention", TypeError, scale="a")
    refused(ops, "paged_attention", ValueError, max_rows=-1)
    refused(ops, "paged_attention", ValueError, max_len=-1)
    refused(ops, "paged_attention", TypeError, max_len=1.5)
    for bad in (-1.0, float("nan"), float("inf")):
        refused(ops, "verify_drafts", ValueError, temperature=bad)
    refused(ops, "verify_drafts", TypeError, temperature=torch.ones(2, device=DEV, dtype=torch.float64))
    refused(ops, "verify_drafts", ValueError, temperature=torch.ones(1, device=DEV))


def test_traced_calls_name_the_entry(monkeypatch, capsys):
    from sequoia_amd.ops import HipOps
    traced = HipOps()
    traced.lib = native._TracedLib(native.load())
    try:
        traced.paged_attention(**attend_args())
        assert "sq-call sq_paged_attention(" in capsys.readouterr().err
    finally:
        fresh = HipOps()                                                 # binds the untraced entries again
        fresh.paged_attention(**attend_args())
    assert "sq-call" not in capsys.readouterr().err
