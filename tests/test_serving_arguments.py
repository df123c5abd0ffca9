"""What Context.q4_gemv_lora, Context.route_scores, Lora and Routing check before
the library is called, case by case, without a GPU: the arguments are CPU
tensors that say they are on the GPU, and the library is one that records its
calls, so every refusal is the named check's and every accepted call gets
through."""
import pytest
import torch

import osm_b200 as osm


class OnGpu:
    """A CPU tensor that reports CUDA device `index`."""

    def __init__(self, t, index=0):
        self.t, self.index = t, index
        self.is_cuda, self.device = True, torch.device("cuda", index)

    def get_device(self):
        return self.index

    def __getitem__(self, i):
        return OnGpu(self.t[i], self.index)

    def __getattr__(self, name):
        return getattr(self.t, name)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(osm, "lib", lambda: lib)
    return lib


@pytest.fixture
def ctx(library):
    c = object.__new__(osm.Context)
    c.h, c.device, c.max_tokens = None, 0, 4
    return c


def projection(**change):
    """Arguments of a projection of 4 tokens, 128 to 32, with three adapters."""
    v = dict(packed=OnGpu(torch.zeros(32, 16, dtype=torch.int32)),
             scales=OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16)),
             biases=OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16)), out_dim=32, in_dim=128,
             x=OnGpu(torch.zeros(4, 128)), tokens=4, y=OnGpu(torch.zeros(4, 32)),
             lora=osm.Lora(OnGpu(torch.zeros(3, 8, 128, dtype=torch.bfloat16)),
                           OnGpu(torch.zeros(3, 32, 8, dtype=torch.bfloat16))),
             adapter=OnGpu(torch.zeros(4, dtype=torch.int32)))
    v.update(change)
    return v


def project(ctx, v):
    ctx.q4_gemv_lora(v["packed"], v["scales"], v["biases"], v["out_dim"], v["in_dim"], v["x"], v["tokens"], v["y"],
                     lora=v["lora"], adapter=v["adapter"])


def test_projection_is_called(ctx, library):
    v = projection()
    project(ctx, v)
    (name, args), = library.calls
    assert name == "osm_q4_gemv_lora"
    assert args[1:4] == tuple(v[k].data_ptr() for k in ("packed", "scales", "biases"))
    assert args[4:11] == (32, 128, 64, v["x"].data_ptr(), 0, 128, 4) and args[13:] == (v["y"].data_ptr(), 32)


@pytest.mark.parametrize("packed,scales", [(torch.int32, torch.bfloat16), (torch.uint32, torch.uint16),
                                           (torch.uint8, torch.uint8), (torch.int32, torch.int16)])
def test_q4_tables_in_the_types_that_hold_them(ctx, library, packed, scales):
    """Words, or the bytes of a slot; bf16, or its bits."""
    n = 4 if packed == torch.uint8 else 1
    m = 2 if scales == torch.uint8 else 1
    tables = dict(packed=OnGpu(torch.zeros(32 * 16 * n, dtype=packed)),
                  scales=OnGpu(torch.zeros(32 * 2 * m, dtype=scales)),
                  biases=OnGpu(torch.zeros(32 * 2 * m + 5, dtype=scales)))
    project(ctx, projection(**tables))
    assert len(library.calls) == 1


@pytest.mark.parametrize("name,table", [
    ("packed", OnGpu(torch.zeros(31, 16, dtype=torch.int32))), ("packed", OnGpu(torch.zeros(32, 16))),
    ("packed", OnGpu(torch.zeros(32 * 16 * 4 - 1, dtype=torch.uint8))),
    ("packed", OnGpu(torch.zeros(32, 32, dtype=torch.int32)[:, ::2])), ("packed", torch.zeros(32, 16, dtype=torch.int32)),
    ("packed", OnGpu(torch.zeros(32, 16, dtype=torch.int32), index=1)),
    ("scales", OnGpu(torch.zeros(32, 1, dtype=torch.bfloat16))), ("scales", OnGpu(torch.zeros(32, 2))),
    ("scales", OnGpu(torch.zeros(32, 2, dtype=torch.float16))), ("scales", torch.zeros(32, 2, dtype=torch.bfloat16)),
    ("biases", OnGpu(torch.zeros(63, dtype=torch.uint16))),
    ("biases", OnGpu(torch.zeros(32, 4, dtype=torch.bfloat16)[:, ::2])),
    ("biases", OnGpu(torch.zeros(32, 2, dtype=torch.bfloat16), index=1))])
def test_q4_tables_that_do_not_hold_the_weights(ctx, library, name, table):
    """Short, of another type, strided, on the CPU or on another device."""
    with pytest.raises(ValueError, match=name):
        project(ctx, projection(**{name: table}))
    assert not library.calls


def route(ctx, tokens=None, routing=None, **change):
    """64 experts, top 8, 4 tokens."""
    v = dict(logits=OnGpu(torch.zeros(4, 64)), ids=OnGpu(torch.zeros(4, 8, dtype=torch.int32)),
             weights=OnGpu(torch.zeros(4, 8)), mass=OnGpu(torch.zeros(4)))
    v.update(change)
    ctx.route_scores(v["logits"], routing or osm.Routing(64, 8), v["ids"], v["weights"], mass=v["mass"], tokens=tokens)


def test_routing_is_called(ctx, library):
    route(ctx)
    route(ctx, tokens=3, logits=OnGpu(torch.zeros(4, 70)[:, :64]))
    assert [(n, a[3:6]) for n, a in library.calls] == [("osm_route_scores", (0, 64, 4)), ("osm_route_scores", (0, 70, 3))]


@pytest.mark.parametrize("tokens", [-1, -2**31, -2**32 + 4, 5])
def test_token_counts(ctx, library, tokens):
    """Counts that are more than the rows, and negative ones, which the
    library's unsigned count would take as billions of rows."""
    with pytest.raises(ValueError, match="rows|token"):
        route(ctx, tokens=tokens)
    with pytest.raises(ValueError, match="rows|token"):
        project(ctx, projection(tokens=tokens))
    assert not library.calls


@pytest.mark.parametrize("field", ["experts", "top_k", "groups", "top_groups"])
@pytest.mark.parametrize("value", [-1, 2**32 + 1])
def test_routing_fields_that_would_wrap(field, value):
    """2**32 + 1 groups are not one group."""
    with pytest.raises(ValueError, match=field):
        osm.Routing(**{**dict(experts=64, top_k=8, groups=2, top_groups=1), field: value})
