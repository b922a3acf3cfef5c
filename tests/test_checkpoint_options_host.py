"""A checkpoint says which of TinyViT's options its network was built with: one that no parameter shows (rotary positions) must not get lost, on the CPU."""
from types import SimpleNamespace

import pytest
import torch


class Optimizer:
    def state_dict(self):
        return {"state": {}, "param_groups": []}

    def load_state_dict(self, sd):
        pass


def agent(tmp_path, **options):
    from semiuhpe_amd.src.agent import SSLAgent
    from semiuhpe_amd.src.tiny_vit import TinyViT21M
    from semiuhpe_amd.src.utils import TrainClock
    a = object.__new__(SSLAgent)
    a.rank, a.clock, a.optimizer = 0, TrainClock(), Optimizer()
    a.config = SimpleNamespace(model_dir=str(tmp_path), exp_name="t", date="t")
    torch.manual_seed(0)
    a.net, a.ema_net = TinyViT21M(**options), TinyViT21M(**options)
    return a


OTHERS = [dict(), dict(rope=True), dict(mlp="gated"), dict(mlp="gated", rope=True)]


def test_checkpoints_load_into_their_own_network_only(tmp_path):
    agents = [agent(tmp_path, **o) for o in OTHERS]
    for i, a in enumerate(agents):
        a.save_ckpt("best")
        saved = torch.load(str(tmp_path / "best.pth"), weights_only=True)
        four = {"clock", "model_state_dict", "model_state_dict_ema", "optimizer_state_dict"}
        assert set(saved) == (four | {"network_options"} if OTHERS[i] else four)
        for j, b in enumerate(agents):
            if i == j:
                b.load_ckpt("best")
            else:
                with pytest.raises(ValueError, match="vit_rope"):
                    b.load_ckpt("best")


def test_dropout_is_no_part_of_it(tmp_path):
    agent(tmp_path, rope=True, drop=0.1).save_ckpt("best")
    agent(tmp_path, rope=True).load_ckpt("best")
