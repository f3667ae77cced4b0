"""Refusals of the operators on device tensors, through C and through Python, without a GPU."""
import ctypes as C

import pytest
import torch

BUF = (C.c_char * 4096)()
AT = (C.addressof(BUF) + 255) & ~255      # never followed: every call below is refused first


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    return device_ops


def refused(b200, rc, exc, words):
    assert rc == {v: k for k, v in b200._STATUS.items()}[exc], (rc, b200.lib().b200_last_error())
    assert words in b200.lib().b200_last_error().decode()


def test_norm_refusals(b200, D):
    good = dict(device=0, stream=None, type=0, x=AT, ldx=64, residual=AT, ldr=64, sum=AT + 256, lds=64, weight=AT, eps=1e-5, q=AT, ldq=64, scales=AT, rows=2, hidden=64)
    for change, exc, words in [
            (dict(type=8), b200.UnsupportedDType, "type 8"), (dict(rows=-1), b200.ShapeMismatch, "rows"), (dict(hidden=0), b200.ShapeMismatch, "hidden"),
            (dict(hidden=65537, ldx=70000, ldq=70000, ldr=70000, lds=70000), b200.ShapeMismatch, "hidden"), (dict(ldx=-1), b200.ShapeMismatch, "negative"), (dict(ldr=-8), b200.ShapeMismatch, "negative"),
            (dict(ldq=1), b200.ShapeMismatch, "overlap"), (dict(lds=0), b200.ShapeMismatch, "overlap"), (dict(x=None), b200.InvalidArgument, "null"),
            (dict(weight=None), b200.InvalidArgument, "null"), (dict(sum=None), b200.InvalidArgument, "null"), (dict(eps=-1.0), b200.InvalidArgument, "eps"),
            (dict(eps=float("nan")), b200.InvalidArgument, "eps"), (dict(sum=AT, lds=65), b200.InvalidArgument, "in place")]:
        refused(b200, D._lib().b200_dev_add_rms_norm_q8(*{**good, **change}.values()), exc, words)
    assert D._lib().b200_dev_add_rms_norm_q8(*{**good, "rows": 0, "x": None}.values()) == 0


def test_values_refusals(b200, D):
    good = dict(device=0, stream=None, type=0, q=AT, ldq=64, s=AT, out=AT, ldo=64, rows=2, n=64)
    for change, exc, words in [(dict(type=9), b200.UnsupportedDType, "type 9"), (dict(rows=-1), b200.ShapeMismatch, "rows"), (dict(n=0), b200.ShapeMismatch, "n"),
                               (dict(ldo=63), b200.ShapeMismatch, "overlap"), (dict(ldq=-1), b200.ShapeMismatch, "negative"), (dict(s=None), b200.InvalidArgument, "null")]:
        refused(b200, D._lib().b200_dev_read_q8(*{**good, **change}.values()), exc, words)
    with pytest.raises(b200.DTypeMismatch):
        D.read_q8(torch.zeros(2, 3), torch.ones(2))
    with pytest.raises(b200.ShapeMismatch):
        D.read_q8(torch.zeros(2, 3, dtype=torch.int8), torch.ones(3))
    with pytest.raises(TypeError):
        D.read_q8([1, 2], torch.ones(2))


def test_product_refusals(b200, D):
    good = dict(device=0, stream=None, type=0, a=AT, lda=64, s=AT, w=AT, ldw=64, ws=AT, bias=None, out=AT, ldo=8, t=2, k=64, n=8)
    for change, exc, words in [
            (dict(type=1000), b200.UnsupportedDType, "type"), (dict(k=0), b200.ShapeMismatch, "shape"), (dict(n=0), b200.ShapeMismatch, "shape"), (dict(t=-3), b200.ShapeMismatch, "shape"),
            (dict(n=(1 << 31) - 1, ldo=1 << 31), b200.ShapeMismatch, "shape"), (dict(t=(1 << 31) - 1), b200.ShapeMismatch, "shape"),
            (dict(k=131072, lda=131072, ldw=131072), b200.ShapeMismatch, "131071"), (dict(lda=48), b200.ShapeMismatch, "overlap"), (dict(ldo=7), b200.ShapeMismatch, "overlap"),
            (dict(a=AT + 8), b200.InvalidArgument, "16 bytes"), (dict(w=AT + 1), b200.InvalidArgument, "16 bytes"), (dict(lda=65), b200.InvalidArgument, "16 bytes"),
            (dict(ldw=72), b200.InvalidArgument, "16 bytes"), (dict(out=None), b200.InvalidArgument, "null"), (dict(ws=None), b200.InvalidArgument, "null")]:
        refused(b200, D._lib().b200_dev_mat_mat_i8(*{**good, **change}.values()), exc, words)


def pages(D, **kw):
    v = dict(data=AT, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    v.update(kw)
    return D.Q4Pages(*v.values())


BAD_PAGES = [(dict(data=None), "InvalidArgument", "null"), (dict(data=AT + 8), "InvalidArgument", "16 bytes"), (dict(head_dim=96), "Unsupported", "head_dim"),
             (dict(page_size=8), "InvalidArgument", "page_size"), (dict(page_size=24), "InvalidArgument", "page_size"), (dict(page_size=2048), "InvalidArgument", "page_size"),
             (dict(n_pages=0), "ShapeMismatch", "pages"), (dict(n_kv_heads=0), "ShapeMismatch", "kv heads")]


def test_append_refusals(b200, D):
    L = D._lib()

    def call(cache=None, **kw):
        a = D.Q4Append(device=0, type=0, q=AT, k=AT, v=AT, q_out=AT, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, q_out_token=256, q_out_head=64, cos_sin=AT,
                       table_rows=10, positions=AT, slots=AT, tokens=3, n_heads=4, rot_dims=64, use_neox=0, cache=cache or pages(D))
        for k, v in kw.items():
            setattr(a, k, v)
        return L.b200_dev_rope_append_q4(C.byref(a))

    for change, exc, words in BAD_PAGES:
        refused(b200, call(pages(D, **change)), getattr(b200, exc), words)
    for change, exc, words in [
            (dict(type=2), b200.UnsupportedDType, "type 2"), (dict(rot_dims=0), b200.ShapeMismatch, "rot_dims"), (dict(rot_dims=63), b200.ShapeMismatch, "rot_dims"),
            (dict(rot_dims=66), b200.ShapeMismatch, "rot_dims"), (dict(tokens=-1), b200.ShapeMismatch, "tokens"), (dict(table_rows=0), b200.ShapeMismatch, "table"),
            (dict(n_heads=0), b200.ShapeMismatch, "heads"), (dict(tokens=1 << 29), b200.ShapeMismatch, "too many"), (dict(slots=None), b200.InvalidArgument, "null"),
            (dict(q_out=None), b200.InvalidArgument, "null"), (dict(cos_sin=None), b200.InvalidArgument, "null"), (dict(q_out_token=512), b200.InvalidArgument, "in place")]:
        refused(b200, call(**change), exc, words)
    refused(b200, L.b200_dev_rope_append_q4(None), b200.InvalidArgument, "null")
    assert call(tokens=0) == 0


def test_read_refusals(b200, D):
    L = D._lib()
    for change, exc, words in BAD_PAGES:
        refused(b200, L.b200_dev_read_q4(0, None, 0, C.byref(pages(D, **change)), AT, 1, AT, AT, None), getattr(b200, exc), words)
    refused(b200, L.b200_dev_read_q4(0, None, 5, C.byref(pages(D)), AT, 1, AT, AT, None), b200.UnsupportedDType, "type 5")
    refused(b200, L.b200_dev_read_q4(0, None, 0, C.byref(pages(D)), None, 1, AT, AT, None), b200.InvalidArgument, "null")
    refused(b200, L.b200_dev_read_q4(0, None, 0, C.byref(pages(D)), AT, 1, AT + 4, AT, None), b200.InvalidArgument, "16 bytes")
    refused(b200, L.b200_dev_read_q4(0, None, 0, C.byref(pages(D)), AT, -1, AT, AT, None), b200.ShapeMismatch, "rows")


def test_attention_refusals(b200, D):
    L = D._lib()

    def struct(cache=None, **kw):
        a = D.Q4Attention(device=0, type=0, q=AT, out=AT, q_token=256, q_head=64, out_token=256, out_head=64, kv_lens=AT, page_table=AT, table_stride=4, tokens=3, table_pages=4, seqs=3,
                          n_heads=4, scale=0.1, cache=cache or pages(D))
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for change, exc, words in BAD_PAGES:
        refused(b200, L.b200_dev_attention_paged_q4(C.byref(struct(pages(D, **change)))), getattr(b200, exc), words)
    for change, exc, words in [
            (dict(type=7), b200.UnsupportedDType, "type 7"), (dict(n_heads=3), b200.ShapeMismatch, "multiple"), (dict(seqs=-1), b200.ShapeMismatch, "negative"),
            (dict(table_stride=-1), b200.ShapeMismatch, "negative"), (dict(table_pages=(1 << 31) // 16 - 1, table_stride=1 << 30), b200.ShapeMismatch, "too many"), (dict(tokens=4), b200.ShapeMismatch, "one token"), (dict(window=-1), b200.InvalidArgument, "window"),
            (dict(tokens=1 << 30, seqs=1 << 30), b200.ShapeMismatch, "too many"), (dict(table_pages=1 << 27, table_stride=1 << 27), b200.ShapeMismatch, "too many"),
            (dict(q=None), b200.InvalidArgument, "null"), (dict(kv_lens=None), b200.InvalidArgument, "null"), (dict(page_table=None), b200.InvalidArgument, "null")]:
        refused(b200, L.b200_dev_attention_paged_q4(C.byref(struct(**change))), exc, words)
    refused(b200, L.b200_dev_attention_paged_q4(None), b200.InvalidArgument, "null")
    refused(b200, L.b200_dev_attention_paged_q4_workspace(C.byref(struct()), None), b200.InvalidArgument, "null")
    need = C.c_size_t(1)
    assert L.b200_dev_attention_paged_q4_workspace(C.byref(struct()), C.byref(need)) == 0
    assert L.b200_dev_attention_paged_q4(C.byref(struct(tokens=0, seqs=0))) == 0
    if need.value:
        for change in (dict(workspace=None, workspace_bytes=1 << 40), dict(workspace=AT, workspace_bytes=need.value - 1), dict(workspace=AT + 16, workspace_bytes=1 << 40)):
            refused(b200, L.b200_dev_attention_paged_q4(C.byref(struct(**change))), b200.InvalidArgument, "workspace")


def test_outputs_whose_rows_overlap_are_refused(b200, D):
    L = D._lib()
    for token, head in ((0, 64), (256, 0), (63, 256), (256, 63), (64, 64), (-256, 64), (255, 64), (64, 191), (1 << 62, 1 << 61)):
        a = D.Q4Append(device=0, type=0, q=AT, k=AT, v=AT, q_out=AT + 4096, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, q_out_token=token, q_out_head=head, cos_sin=AT,
                       table_rows=10, positions=AT, slots=AT, tokens=3, n_heads=4, rot_dims=64, use_neox=0, cache=pages(D))
        refused(b200, L.b200_dev_rope_append_q4(C.byref(a)), b200.ShapeMismatch, "overlap")
        o = D.Q4Attention(device=0, type=0, q=AT, out=AT, q_token=256, q_head=64, out_token=token, out_head=head, kv_lens=AT, page_table=AT, table_stride=4, tokens=3, table_pages=4, seqs=3,
                          n_heads=4, scale=0.1, cache=pages(D))
        refused(b200, L.b200_dev_attention_paged_q4(C.byref(o)), b200.ShapeMismatch, "overlap")


def test_python_refusals(b200, D):
    f32, i8 = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8)
    one = torch.ones(64)
    with pytest.raises(b200.InvalidArgument, match="CUDA"):
        D.add_rms_norm_q8(f32, one, 1e-5)
    with pytest.raises(b200.UnsupportedDType):
        D.add_rms_norm_q8(f32.double(), one, 1e-5)
    with pytest.raises(b200.DTypeMismatch, match="weight"):
        D.add_rms_norm_q8(f32, one.half(), 1e-5)
    with pytest.raises(b200.DTypeMismatch, match="residual"):
        D.add_rms_norm_q8(f32, one, 1e-5, residual=f32.half())
    with pytest.raises(b200.ShapeMismatch, match="weight"):
        D.add_rms_norm_q8(f32, one[:63], 1e-5)
    with pytest.raises(b200.ShapeMismatch, match="x"):
        D.add_rms_norm_q8(f32.T, torch.ones(4), 1e-5)
    with pytest.raises(b200.ShapeMismatch):
        D.add_rms_norm_q8(f32[0], one, 1e-5)
    with pytest.raises(b200.InvalidArgument, match="residual"):
        D.add_rms_norm_q8(f32, one, 1e-5, sum_out=f32)
    with pytest.raises(b200.Unsupported, match="gradient"):
        D.add_rms_norm_q8(f32, one.clone().requires_grad_(), 1e-5)
    s = torch.ones(4)
    with pytest.raises(b200.ShapeMismatch, match="w"):
        D.mat_mat_i8(i8, s, i8[:, :32], s)
    with pytest.raises(b200.ShapeMismatch, match="a_scales"):
        D.mat_mat_i8(i8, s[:3], i8, s)
    with pytest.raises(b200.DTypeMismatch):
        D.mat_mat_i8(f32, s, i8, s)
    with pytest.raises(b200.UnsupportedDType):
        D.mat_mat_i8(i8, s, i8, s, dtype=torch.int32)
    with pytest.raises(b200.InvalidArgument, match="CUDA"):
        D.mat_mat_i8(i8, s, i8, s)
    k, v, slots, pos = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.long), torch.zeros(3, dtype=torch.int32)
    cs, pg = D.rotary_table(8, 64, device="cpu"), D.q4_pages(2, 2, 64, 16, device="cpu")
    assert pg.shape == (2, 2, 16 * 72)
    for bad, exc in [(dict(k=k[0]), b200.ShapeMismatch), (dict(v=v[:, :1]), b200.ShapeMismatch), (dict(v=v.half()), b200.DTypeMismatch), (dict(slots=slots.int()), b200.DTypeMismatch),
                     (dict(positions=pos.long()), b200.DTypeMismatch), (dict(slots=slots[:2]), b200.ShapeMismatch), (dict(pages=pg[:, :, :100]), b200.ShapeMismatch),
                     (dict(pages=pg[:, :1].contiguous()), b200.ShapeMismatch), (dict(pages=pg.float()), b200.DTypeMismatch), (dict(cos_sin=cs.double()), b200.DTypeMismatch),
                     (dict(q=torch.zeros(2, 4, 64)), b200.ShapeMismatch), (dict(q=torch.zeros(3, 4, 32)), b200.ShapeMismatch), (dict(), b200.InvalidArgument)]:
        args = dict(q=None, k=k, v=v, cos_sin=cs, positions=pos, pages=pg, slots=slots)
        args.update(bad)
        with pytest.raises(exc):
            D.rope_append_q4(**args)
    q, table, lens = torch.zeros(2, 4, 64), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad, exc in [(dict(q=q[0]), b200.ShapeMismatch), (dict(q=q.double()), b200.UnsupportedDType), (dict(page_table=table.long()), b200.DTypeMismatch), (dict(page_table=table[0]), b200.ShapeMismatch),
                     (dict(kv_lens=lens[:1]), b200.ShapeMismatch), (dict(q_starts=lens), b200.ShapeMismatch), (dict(scale=float("inf")), b200.InvalidArgument),
                     (dict(out=q.half()), b200.DTypeMismatch), (dict(), b200.InvalidArgument)]:
        args = dict(q=q, pages=pg, page_table=table, kv_lens=lens)
        args.update(bad)
        with pytest.raises(exc):
            D.attention_paged_q4(**args)
    with pytest.raises(b200.DTypeMismatch):
        D.read_q4(pg, slots.int(), 64)


def test_rotary_table(D):
    t = D.rotary_table(100, 8, base=500.0, scale=2.0, device="cpu").double()
    for p in (0, 1, 99):
        for i in range(4):
            a = p / 2.0 * 500.0 ** (-2 * i / 8)
            assert abs(t[p, i] - torch.tensor(a).double().cos()) < 1e-6 and abs(t[p, 4 + i] - torch.tensor(a, dtype=torch.float64).sin()) < 1e-6
