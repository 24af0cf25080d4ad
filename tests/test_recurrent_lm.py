"""The recurrent language model through the public API on the host: training under strategies, checkpoints of the list optimizer's moments, and
answering in 8 bits."""
import os

import pytest
import torch

from autodist_b200 import AutoDist
from autodist_b200 import strategy as S
from autodist_b200.autodist import _reset_default_autodist
from autodist_b200.checkpoint.saver import Saver
from autodist_b200.models.recurrent_lm import RecurrentLM, RecurrentLMConfig, cyclic_tokens
from autodist_b200.optim import ListAdamW
from autodist_b200.resource_spec import ResourceSpec

CONFIG = RecurrentLMConfig(vocab_size=60, width=32, units=48, layers=2)


class _Session:
    def __init__(self, builder, bits, seed=3):
        _reset_default_autodist()
        os.environ["AUTODIST_IS_TESTING"] = "True"
        self.ad = AutoDist(resource_spec=ResourceSpec.local(num_cpus=1), strategy_builder=builder)
        data = cyclic_tokens(6, 12, CONFIG.vocab_size)
        self.scope = self.ad.scope()
        self.scope.__enter__()
        torch.manual_seed(seed)
        self.model = RecurrentLM(CONFIG)
        phs = {k: self.ad.placeholder((None, 12), torch.int64, name=k) for k in data}
        loss = self.model(**phs)
        train_op = ListAdamW(self.model.parameters(), lr=5e-3, state_bits=bits).minimize(loss)
        self.saver = Saver()
        self.sess = self.ad.create_distributed_session()
        self.step = lambda: float(self.sess.run([loss, train_op], {phs[k]: data[k] for k in phs})[0])

    def done(self):
        self.sess.close()
        self.scope.__exit__(None, None, None)
        _reset_default_autodist()


@pytest.mark.parametrize("builder", [S.AllReduce, S.PartitionedPS, S.PS])
@pytest.mark.parametrize("bits", [8, 32])
def test_trains_and_resumes_from_a_checkpoint(builder, bits, tmp_path):
    s = _Session(builder(), bits)
    losses = [s.step() for _ in range(6)]
    assert losses[-1] < losses[0]
    path = s.saver.save(s.sess, str(tmp_path / "model"), global_step=6)
    expected = [s.step() for _ in range(3)]
    s.done()
    again = _Session(builder(), bits, seed=9)
    again.saver.restore(again.sess, path)
    got = [again.step() for _ in range(3)]
    again.done()
    # 32 bits go on as they were; 8 bits come back as they were held, but for values that their block's largest moves by a rounding
    assert got == pytest.approx(expected, rel=1e-5 if bits == 32 else 2e-2)


def test_eight_bits_answer_as_the_model_does():
    torch.manual_seed(0)
    model = RecurrentLM(CONFIG)
    data = cyclic_tokens(8, 24, CONFIG.vocab_size)
    opt = ListAdamW(model.parameters(), lr=1e-2)
    for _ in range(40):
        opt.zero_grad()
        model(data["x"], data["y"]).backward()
        opt.step()
    answer = model.answerer()
    logits, states = answer(data["x"][:, :10])
    for t in range(10, 20):                         # the prompt in one go, the rest a token at a time
        assert torch.equal(logits.argmax(-1), data["x"][:, t])
        logits, states = answer(data["x"][:, t:t + 1], states)
    whole, _ = answer(data["x"][:, :20])
    assert torch.allclose(whole.float(), logits.float(), atol=0.05 * float(whole.float().abs().max()))
