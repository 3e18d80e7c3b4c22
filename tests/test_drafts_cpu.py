"""The operators of drafted tokens without a GPU: what they refuse, in Python and at the C ABI (before any launch), the shapes of
their registered ops under a tracer, and the host's own oracle against the definition of what it decides."""

from __future__ import annotations

import ctypes
import itertools
import os
import random
import re
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from kernelforge import _lib, build, ops

from draft_cases import ancestors_of, positions_of, verify_on_host
from test_paged_cpu import _struct, attention_args

I32 = torch.int32


def zeros(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def tree_args():
    return dict(parents=zeros(6), cu_new=zeros(3), seq_lens=zeros(2))


@pytest.mark.parametrize("change,error,match", [
    (dict(parents=zeros(6, dtype=torch.int64)), ValueError, "parents"), (dict(parents=zeros(2, 3)), ValueError, "parents"),
    (dict(parents=zeros(12)[::2]), ValueError, "parents"), (dict(cu_new=zeros(2)), ValueError, "cu_new"),
    (dict(seq_lens=zeros(2, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(seq_lens=zeros(0), cu_new=zeros(1)), ValueError, "at least one request"), (dict(), RuntimeError, "CUDA device"),
])
def test_draft_trees_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.draft_trees(**{**tree_args(), **change})


def attend_args(**kw):
    return {**attention_args(**kw), "ancestors": torch.zeros(6, dtype=torch.int64, device=kw.get("device", "cpu"))}


@pytest.mark.parametrize("change,error,match", [
    (dict(ancestors=zeros(6)), ValueError, "ancestors"), (dict(ancestors=zeros(7, dtype=torch.int64)), ValueError, "ancestors"),
    (dict(ancestors=zeros(12, dtype=torch.int64)[::2]), ValueError, "ancestors"),
    (dict(q=torch.zeros(6, 4, 64)), TypeError, "fp16 or bf16"), (dict(q=torch.zeros(6, 256, dtype=torch.float16)), TypeError, "3-D"),
    (dict(q=torch.zeros(6, 3, 64, dtype=torch.float16)), ValueError, "must divide"),
    (dict(cache_v=torch.zeros(5, 2, 16, 64)), TypeError, "cache_v must have the type"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "block_table"), (dict(cu_new=zeros(2)), ValueError, "cu_new"),
    (dict(max_new=0), ValueError, "max_new"), (dict(scale=2.4e38), ValueError, "at most 2.35e38"),
    (dict(out=torch.zeros(6, 1, 64, dtype=torch.float16).expand(6, 4, 64)), ValueError, "none of them 0"),
    (dict(out=torch.zeros(6, 4, 64, dtype=torch.float16, requires_grad=True)), RuntimeError, "inference only"),
    (dict(), RuntimeError, "CUDA device"),
])
def test_paged_tree_attention_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.paged_tree_attention(**{**attend_args(), **change})
    with pytest.raises(ValueError, match="paged_tree_attention needs at least one request"):
        ops.paged_tree_attention(**attend_args(b=0))


def verify_args(sampled=True, drawn=True):
    args = dict(tokens=zeros(6, dtype=torch.int64), parents=zeros(6), cu_new=zeros(3), target=torch.zeros(6, 50))
    if sampled:
        args.update(accept_uniforms=torch.zeros(6), sample_uniforms=torch.zeros(2))
    if drawn:
        args.update(draft=torch.zeros(6, 50))
    return args


@pytest.mark.parametrize("change,error,match", [
    (dict(tokens=zeros(6)), ValueError, "tokens"), (dict(tokens=zeros(5, dtype=torch.int64)), ValueError, "tokens"),
    (dict(parents=zeros(6, dtype=torch.int64)), ValueError, "parents"), (dict(parents=zeros(7)), ValueError, "parents"),
    (dict(cu_new=zeros(3, dtype=torch.int64)), ValueError, "cu_new"), (dict(cu_new=zeros(1)), ValueError, "at least one request"),
    (dict(target=torch.zeros(6)), TypeError, "target"), (dict(target=torch.zeros(6, 50, dtype=torch.float16)), TypeError, "target"),
    (dict(target=torch.zeros(6, 50, dtype=torch.float64)), TypeError, "target"),
    (dict(target=torch.zeros(6, 0), draft=torch.zeros(6, 0)), ValueError, "one token"),
    (dict(accept_uniforms=torch.zeros(5)), ValueError, "accept_uniforms"),
    (dict(accept_uniforms=torch.zeros(6, dtype=torch.float64)), ValueError, "accept_uniforms"),
    (dict(sample_uniforms=torch.zeros(6)), ValueError, "sample_uniforms"), (dict(sample_uniforms=None), ValueError, "come together"),
    (dict(accept_uniforms=None), ValueError, "come together"),
    (dict(accept_uniforms=None, sample_uniforms=None), ValueError, "draft needs"),
    (dict(draft=torch.zeros(6, 49)), ValueError, "draft must be"), (dict(draft=torch.zeros(6, 50).half()), ValueError, "draft must be"),
    (dict(max_new=0), ValueError, "max_new"), (dict(max_new=-1), ValueError, "max_new"), (dict(), RuntimeError, "CUDA device"),
])
def test_verify_drafts_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.verify_drafts(**{**verify_args(), **change})


def test_scores_of_other_types():
    for dtype in (torch.float16, torch.bfloat16):
        with pytest.raises(RuntimeError, match="CUDA device"):
            ops.verify_drafts(**{**verify_args(False, False), "target": torch.zeros(6, 50, dtype=dtype)})
    with pytest.raises(TypeError, match="target"):
        ops.verify_drafts(**{**verify_args(False, False), "target": torch.zeros(6, 50, dtype=torch.int32)})


def keep_args(caches=None):
    return dict(caches=torch.zeros(4, 5, 2, 16, 64, dtype=torch.float16) if caches is None else caches, block_table=zeros(2, 3),
                context_lens=zeros(2), seq_lens=zeros(2), counts=zeros(2), path=zeros(2, 64), free_pages=zeros(9),
                free_count=zeros(1))


H = dict(dtype=torch.float16)
CACHE = torch.zeros(4, 5, 2, 16, 64, **H)


@pytest.mark.parametrize("change,error,match", [
    (dict(caches=torch.zeros(4, 5, 2, 16, 64)), TypeError, "fp16 or bf16"), (dict(caches=[]), ValueError, "at least one cache"),
    (dict(caches=torch.zeros(2, 16, 64, **H)), ValueError, "num_pages"), (dict(caches=torch.zeros(0, 5, 2, 16, 64, **H)), ValueError, "empty"),
    (dict(caches=torch.zeros(4, 5, 2, 24, 64, **H)), ValueError, "power of two"),
    (dict(caches=torch.zeros(4, 5, 2, 16, 60, **H)), ValueError, "multiple of 8"),
    (dict(caches=torch.zeros(4, 5, 2, 16, 68, **H)[..., :64]), ValueError, "multiples of 8"),
    (dict(caches=torch.zeros(4, 1, 2, 16, 64, **H).expand(4, 5, 2, 16, 64)), ValueError, "none of them 0"),
    (dict(caches=torch.zeros(3, 4, 5, 2, 16, 64, **H)[:, :2]), ValueError, "leading dimensions"),
    (dict(caches=[torch.zeros(5, 2, 16, 64, **H), torch.zeros(5, 2, 16, 64)]), TypeError, "fp16 or bf16"),
    (dict(caches=[CACHE, CACHE]), ValueError, "different arrays"), (dict(caches=[CACHE, CACHE[0]]), ValueError, "different arrays"),
    (dict(block_table=zeros(2, 3, dtype=torch.int64)), ValueError, "block_table"), (dict(block_table=zeros(0, 3)), ValueError, "at least one"),
    (dict(context_lens=zeros(3)), ValueError, "context_lens"), (dict(seq_lens=zeros(2, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(counts=zeros(1)), ValueError, "counts"), (dict(path=zeros(2, 65)), ValueError, "path"), (dict(path=zeros(2, 0)), ValueError, "path"),
    (dict(path=zeros(3, 64)), ValueError, "path"), (dict(path=zeros(2, 128)[:, ::2]), ValueError, "path"),
    (dict(free_count=None), ValueError, "come together"), (dict(free_pages=None), ValueError, "come together"),
    (dict(free_count=zeros(2)), ValueError, "free_count"), (dict(free_pages=zeros(3, 3)), ValueError, "free_pages"),
    (dict(), RuntimeError, "CUDA device"),
])
def test_keep_drafts_refusals(change, error, match):
    with pytest.raises(error, match=match):
        ops.keep_drafts(**{**keep_args(), **change})


@pytest.mark.parametrize("op,args,name", [(ops.paged_tree_attention, attend_args, "q"), (ops.verify_drafts, verify_args, "target"),
                                          (ops.verify_drafts, verify_args, "draft"), (ops.keep_drafts, keep_args, "caches")])
def test_gradients_and_transforms_are_refused(op, args, name):
    a = args()
    a[name] = a[name].requires_grad_()
    with pytest.raises(RuntimeError, match="inference only"):
        op(**a)
    a = args()
    x = a.pop(name)
    with pytest.raises(RuntimeError, match="cannot be transformed"):
        torch.func.vmap(lambda y: op(**{name: y}, **a))(x[None])


def test_shapes_under_a_tracer():
    with FakeTensorMode(), torch.no_grad():
        def on_gpu(args):
            return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in args.items()}

        tree = ops.draft_trees(**on_gpu(tree_args()))
        assert tree.ancestors.shape == tree.positions.shape == (6,) and tree.positions.dtype == torch.int64
        a = attend_args(device="cuda")
        assert ops.paged_tree_attention(**a).shape == (6, 4, 64)
        with pytest.raises(RuntimeError, match="no traceable form"):
            ops.paged_tree_attention(**a, out=torch.empty_like(a["q"]))
        for args in (verify_args(), verify_args(True, False), verify_args(False, False)):
            done = ops.verify_drafts(**on_gpu(args), max_new=7)
            assert [tuple(t.shape) for t in done] == [(2,), (2, 7), (2, 7)] and done.tokens.dtype == torch.int64
        kept = ops.keep_drafts(**on_gpu(keep_args()))
        assert kept.context_lens.shape == (2,) and kept.free_count.shape == (1,)


def _err(status, match):
    assert status != 0
    assert re.search(match, _lib.last_error()), _lib.last_error()


def struct(cls, **change):
    values = {_lib.VerifyDraftsArgs: dict(vocab=50, width=64, mode=0, tokens_count=4), _lib.KeepDraftsArgs: dict(arrays=4, width=64)}
    return _struct(cls, **{**values.get(cls, {}), **change})


@pytest.mark.parametrize("change,match", [(dict(parents=None), "non-null"), (dict(positions=None), "non-null"),
                                          (dict(tokens=-1), "tokens >= 0"), (dict(seqs=0), "seqs >= 1"), (dict(seqs=65536), "up to 65535")])
def test_draft_trees_abi(change, match):
    _err(_lib.load().kf_draft_trees(ctypes.byref(struct(_lib.DraftTreesArgs, **change)), None), match)


@pytest.mark.parametrize("change,match", [(dict(q=None), "non-null"), (dict(block_size=48), "power of two"), (dict(max_new=-1), "max_new"),
                                          (dict(k_page=4), "multiples of 8"), (dict(scale=0.0), "scale")])
def test_paged_tree_attention_abi(change, match):
    args = struct(_lib.PagedAttentionArgs, **change)
    _err(_lib.load().kf_paged_tree_attention(ctypes.byref(args), 0x1000, 0x1000, 1 << 40, None), match)


@pytest.mark.parametrize("change,match", [
    (dict(tokens=None), "non-null"), (dict(path=None), "non-null"), (dict(mode=1, sample_u=None), "non-null"),
    (dict(mode=1, accept_u=None), "non-null"), (dict(mode=2, draft=None), "non-null"), (dict(mode=3), "mode"), (dict(mode=-1), "mode"),
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"), (dict(width=0), "1 to 64"), (dict(width=65), "1 to 64"),
    (dict(seqs=0), "seqs"), (dict(seqs=65536), "up to 65535"), (dict(tokens_count=-1), "tokens"), (dict(tokens_count=1 << 23), "more than"),
    (dict(dtype=3), "dtype|scores"), (dict(mode=1, dtype=1), "scores"), (dict(target_row=-1), "negative"),
])
def test_verify_drafts_abi(change, match):
    change = {"dtype": 0, **change}
    _err(_lib.load().kf_verify_drafts(ctypes.byref(struct(_lib.VerifyDraftsArgs, **change)), 0x1000, 1 << 40, None), match)


def test_verify_workspaces():
    lib = _lib.load()
    for mode in (0, 1, 2):
        args = struct(_lib.VerifyDraftsArgs, dtype=0, mode=mode, vocab=100000)
        need = lib.kf_verify_drafts_workspace_bytes(ctypes.byref(args))
        assert need > 0
        _err(lib.kf_verify_drafts(ctypes.byref(args), 0x1000, need - 1, None), "workspace too small")
        _err(lib.kf_verify_drafts(ctypes.byref(args), None, need, None), "workspace too small")
        _err(lib.kf_verify_drafts(ctypes.byref(args), 0x1008, need, None), "16-byte aligned")


@pytest.mark.parametrize("change,match", [
    (dict(caches=None), "non-null"), (dict(counts=None), "non-null"), (dict(free_pages=None), "non-null"), (dict(free_left=None), "non-null"),
    (dict(caches=0x1008), "16-byte"), (dict(arrays=0), "arrays"), (dict(num_pages=0), "num_pages"), (dict(head_dim=12), "multiple of 8"),
    (dict(width=65), "1 to 64"), (dict(block_size=8), "power of two"), (dict(table_width=1 << 28), "too long"),
    (dict(seqs=1 << 16, table_width=1 << 15), "too long"), (dict(page_stride=4), "multiples of 8"),
    (dict(kept_lens=0x1230, context_lens=0x1230), "of their own"), (dict(free_left=0x1230, free_count=0x1230), "of their own"),
])
def test_keep_drafts_abi(change, match):
    _err(_lib.load().kf_keep_drafts(ctypes.byref(struct(_lib.KeepDraftsArgs, **change)), None), match)


def test_null_arguments_and_empty_batches():
    lib = _lib.load()
    for fn in (lib.kf_draft_trees, lib.kf_keep_drafts):
        _err(fn(None, None), "args must be non-null")
    _err(lib.kf_verify_drafts(None, None, 0, None), "args must be non-null")
    _err(lib.kf_paged_tree_attention(None, None, None, 0, None), "args must be non-null")
    _err(lib.kf_paged_tree_attention(ctypes.byref(struct(_lib.PagedAttentionArgs)), None, 0x1000, 1 << 40, None), "non-null")
    assert lib.kf_verify_drafts_workspace_bytes(None) == lib.kf_paged_tree_attention_workspace_bytes(None) == 0
    assert lib.kf_draft_trees(ctypes.byref(struct(_lib.DraftTreesArgs, tokens=0, parents=None)), None) == 0


@pytest.mark.parametrize("cls,pack", [(_lib.DraftTreesArgs, _lib.pack_draft_trees), (_lib.VerifyDraftsArgs, _lib.pack_verify_drafts),
                                      (_lib.KeepDraftsArgs, _lib.pack_keep_drafts)])
def test_packed_arguments_are_the_structure(cls, pack):
    values = [(1 << 40) + i if kind is not ctypes.c_int else i - 3 for i, (_, kind) in enumerate(cls._fields_)]
    assert pack(*values) == bytes(cls(*values))
    values[-1] = 1 << 32
    with pytest.raises(ValueError, match="more than one call takes"):
        pack(*values)


def test_words_and_positions_on_the_host():
    parents = [-1, 0, 1, 1, 3, -1, 5, 9]
    assert ancestors_of(parents) == [1, 3, 7, 11, 27, 32, 96, 128]
    assert positions_of(parents, 10) == [10, 11, 12, 12, 13, 10, 11, 10]
    assert ancestors_of([-1] + list(range(65)))[63:] == [-1, 0, 0]


def test_the_walk_on_the_host():
    """By hand: p of node 0 is (0.5, 0.25, 0.25); its children are tokens 1 and 2."""
    p = torch.tensor([[0.5, 0.25, 0.25]] * 3)
    call = dict(tokens=[0, 1, 2], parents=[-1, 0, 0], lens=[3], target=p, sample=torch.tensor([0.6]), width=3)
    # Given: 0.2 < 0.25 takes the first; 0.3 does not, then 0.3 x 0.75 < 0.25 the second, 0.34 x 0.75 not.
    assert verify_on_host(accept=torch.tensor([0, 0.2, 0.9]), **call)[1] == [[0, 1, -1]]
    assert verify_on_host(accept=torch.tensor([0, 0.3, 0.3]), **call)[1] == [[0, 2, -1]]
    counts, path, emitted = verify_on_host(accept=torch.tensor([0, 0.3, 0.34]), **call)
    assert (counts, path, emitted) == ([1], [[0, -1, -1]], [[0, -1, -1]])  # only token 0 is left
    # Drawn from (0, 0.5, 0.5): p / q = 0.5; after one rejection f = (0.5, 0, 0), so no second sibling passes.
    q = torch.tensor([[0.0, 0.5, 0.5]] * 3)
    assert verify_on_host(accept=torch.tensor([0, 0.49, 0.0]), draft=q, **call)[1] == [[0, 1, -1]]
    assert verify_on_host(accept=torch.tensor([0, 0.51, 0.0]), draft=q, **call)[2] == [[0, -1, -1]]


def test_layouts_that_meet():
    """Against all places of small arrays, one by one; and a search that is given up counts as a meeting."""
    rng, hits = random.Random(0), 0

    def places(shape, stride):
        return {sum(i * s for i, s in zip(index, stride)) for index in itertools.product(*map(range, shape))}

    for _ in range(3000):
        a, b = (tuple(zip(*[(rng.randrange(1, 4), rng.choice(strides)) for _ in range(rng.randrange(1, 5))]))
                for strides in ((1, 2, 3, 4, 6, 8, 12, 24, 5), (1, 2, 3, 4, 6, 8, 12, 24, 7)))
        apart = rng.randrange(-10, 60)
        want = bool(places(*a) & {p + apart for p in places(*b)})
        assert ops._layouts_meet(a, b, apart) == want, (a, b, apart)
        hits += want
    assert 300 < hits < 2700
    wide = ((5000, 22, 4, 16, 64), (22 * 8192, 8192, 1024, 64, 1))
    assert not ops._layouts_meet(wide, wide, 4096) and ops._layouts_meet(wide, wide, 8192)
    assert ops._layouts_meet(wide, wide, 4096, most_steps=1)


@pytest.mark.parametrize("views", [
    lambda c: [c, c[1:]], lambda c: [c[3], c[1:]], lambda c: [c[:3], c[2:]], lambda c: [c[:, :4], c[:, 3:]],
    lambda c: [c[0], c.view(-1)[64:64 + c[0].numel()].view(c[0].shape)], lambda c: [c[..., :64], c[2:3, ..., 32:]],
    lambda c: [c[0], c[2], c[3], c[2:3]],
])
def test_caches_that_share_places(views):
    with pytest.raises(ValueError, match="different arrays"):
        ops.keep_drafts(**keep_args(views(torch.zeros(4, 5, 2, 16, 64, dtype=torch.float16))))


@pytest.mark.parametrize("views", [
    lambda c: list(c), lambda c: [c[:1], c[1], c[2:]], lambda c: [c[::2], c[1::2]], lambda c: [c[:, :3], c[:, 3:]],
    lambda c: [c[..., :32], c[..., 32:]], lambda c: [c[:, :, :1], c[:, :, 1:]], lambda c: list(c.transpose(0, 1)),
])
def test_views_of_one_tensor_that_share_no_place(views):
    """Past the checks, as far as the device."""
    with pytest.raises(RuntimeError, match="CUDA device"):
        ops.keep_drafts(**keep_args(views(torch.zeros(4, 5, 2, 16, 64, dtype=torch.float16))))


def test_caches_of_several_block_sizes():
    """One table cannot be of pages of 16 and of 32 tokens."""
    with pytest.raises(ValueError, match="one block size"):
        ops.keep_drafts(**keep_args([CACHE, torch.zeros(4, 5, 2, 32, 64, **H)]))


def test_a_list_under_a_tracer():
    """One registered op, whose shapes are those of the lengths; what shares places is refused where it runs."""
    with FakeTensorMode(), torch.no_grad():
        args = {k: v.cuda() for k, v in keep_args().items()}
        args["caches"] = [args["caches"], torch.zeros(5, 2, 16, 64, **H).cuda()]
        kept = ops.keep_drafts(**args)
        assert kept.context_lens.shape == (2,) and kept.free_count.shape == (1,)
    cache, rest = CACHE.clone(), list(keep_args().values())[1:]
    with pytest.raises(ValueError, match="different arrays"):
        torch.ops.kernelforge.keep_listed_drafts([cache, cache[1:]], *rest)


def test_sums_are_handed_on_as_one_processor_orders_them():
    """The hand-over between workgroups leaves out fences that the language asks for: a build for another processor fails."""
    source = build.SRC_DIR / "kf_drafts.hip"
    for arch, fails in (("gfx90a", True), (build.ARCH, False)):
        done = subprocess.run([build.hipcc(), "-E", "--cuda-device-only", f"--offload-arch={arch}", "-std=c++17", "-I",
                               str(build.INCLUDE_DIR), "-I", str(build.SRC_DIR), str(source), "-o", os.devnull],
                              capture_output=True, text=True)
        assert (done.returncode != 0) == fails == ("need a release and an acquire" in done.stderr), done.stderr[-2000:]
