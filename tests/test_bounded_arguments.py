"""The tensors that the bounded cache's calls turn down before any address goes to a
kernel (no GPU: the objects have no handle, and their device is none of the tensors', or
for tensors of the right device, that of CPU tensors)."""
import numpy as np
import pytest
import torch

import kvcu

R, P, W, H = 512, 64, 576, 4
NONE = -1  # what a CPU tensor gives as its device


def bare(cls, device, **members):
    x = cls.__new__(cls)
    x._h, x.device = None, device
    for k, v in members.items():
        setattr(x, k, v)
    return x


def real(*shape):
    return torch.zeros(*shape)


def whole(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def calls(device):
    """Name -> (call of keyword tensors, tensors that it takes)."""
    pool = bare(kvcu.DevicePool, device)
    ws = bare(kvcu.DecodeWorkspace, device)
    cache = bare(kvcu.KVCache, device, kv_rank=R, rope_dim=P, n_layers=2)
    return {
        "evict_select": (lambda **t: pool.evict_select(budget=8, n_sink=1, n_recent=1, **t),
                         dict(mass=real(2, 3, 20), lens=whole(3), keep=whole(2, 3, 8), counts=whole(3), seq_ids=whole(3))),
        "evict_compact": (lambda **t: pool.evict_compact(0, **t),
                          dict(table_offsets=whole(4), tables=whole(6), keep=whole(2, 3, 8), counts=whole(3),
                               mass=real(2, 3, 20), lens=whole(3), seq_ids=whole(3))),
        "attn_mass": (lambda **t: ws.attn_mass(pool, 0, scale=1.0, **t),
                      dict(q=real(3, 2, H, W), lse=real(3, 2, H), table_offsets=whole(4), tables=whole(6), lens=whole(3),
                           mass=real(3, 20), old_lens=whole(3), seq_ids=whole(3))),
        "attnMass_dev": (lambda **t: cache.attnMass_dev(0, [0, 1, 2], scale=1.0, **t),
                         dict(q_dev=real(3, 2, H, W), lse_dev=real(3, 2, H), mass_dev=real(3, 20))),
        "evict_dev": (lambda **t: cache.evict_dev([0, 1, 2], 8, **t),
                      dict(mass_dev=real(2, 3, 20), keep_dev=whole(2, 3, 8))),
        "mla_step_rope_dev": (lambda **t: cache.mla_step_rope_dev(0, [0, 1], [3, 4], kvcu.Rope(P), eps=1e-6, qk_nope=8,
                                                                  v_dim=8, scale=1.0, **t),
                              dict(q=real(2, H, 8 + P), kv_a=real(2, W), norm_w=real(R), k_b=real(H * 8, R),
                                   v_b=real(H * 8, R), attn=real(2, H, 8), q_abs=real(2, H, W), lse=real(2, H))),
        "mlaDecodeLse_dev": (lambda **t: cache.mlaDecodeLse_dev(0, [0, 1], scale=1.0, **t),
                             dict(q_dev=real(2, H, W), out_dev=real(2, H, R), lse_dev=real(2, H))),
        "mlaAttentionBatchLse_dev": (lambda **t: cache.mlaAttentionBatchLse_dev(0, 0, 5, scale=1.0, **t),
                                     dict(q_dev=real(2, H, W), out_dev=real(2, H, R), lse_dev=real(2, H))),
    }


EACH = [(name, t) for name, (_, tensors) in calls(NONE).items() for t in tensors]


@pytest.mark.parametrize("name", calls(NONE))
def test_good_tensors_reach_the_library(name):
    call, tensors = calls(NONE)[name]
    with pytest.raises(kvcu.KVCudaError) as e:  # where there is no handle
        call(**tensors)
    assert e.value.name == "InvalidArgument"


@pytest.mark.parametrize("name,which", EACH)
def test_a_tensor_of_another_device(name, which):
    call, tensors = calls(0)[name]
    with pytest.raises(ValueError, match="cuda:0"):  # all of them on the CPU
        call(**tensors)
    call, tensors = calls(NONE)[name]
    tensors[which] = tensors[which].to("meta")
    with pytest.raises((ValueError, RuntimeError)):
        call(**tensors)


@pytest.mark.parametrize("name,which", EACH)
def test_a_tensor_of_another_type(name, which):
    """The other kind of 32 bits, and 64 bits."""
    call, tensors = calls(NONE)[name]
    for kind in (torch.int32, torch.int64) if tensors[which].dtype == torch.float32 else (torch.float32, torch.int64):
        bad = dict(tensors)
        bad[which] = tensors[which].to(kind)
        with pytest.raises(ValueError):
            call(**bad)


@pytest.mark.parametrize("name,which", EACH)
def test_a_tensor_with_gaps(name, which):
    call, tensors = calls(NONE)[name]
    t = tensors[which]
    tensors[which] = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype)[..., ::2]
    with pytest.raises(ValueError):
        call(**tensors)


# only the device knows how many tables there are; fewer sequences than entries may be there where ids choose
# them; fewer queries of a prompt are another call
OPEN = {("evict_select", "lens"), ("evict_compact", "tables"), ("evict_compact", "table_offsets"), ("attn_mass", "tables"),
        ("attn_mass", "lens"), ("mlaAttentionBatchLse_dev", "q_dev")}


@pytest.mark.parametrize("name,which", [x for x in EACH if x not in OPEN])
def test_a_tensor_that_is_too_short(name, which):
    call, tensors = calls(NONE)[name]
    tensors[which] = tensors[which][:-1].contiguous()
    with pytest.raises(ValueError):
        call(**tensors)


def test_other_numbers_of_dimensions():
    call, tensors = calls(NONE)["attnMass_dev"]
    with pytest.raises(ValueError):
        call(**{**tensors, "mass_dev": real(3, 5, 4)})
    call, tensors = calls(NONE)["attn_mass"]
    with pytest.raises(ValueError):
        call(**{**tensors, "mass": real(3, 5, 4)})


def test_other_numbers_of_sequences():
    cache = bare(kvcu.KVCache, NONE, kv_rank=R, rope_dim=P, n_layers=2)
    with pytest.raises(ValueError):
        cache.mlaDecodeLse_dev(0, np.array([0]), real(2, H, W), 1.0, real(2, H, R), real(2, H))
