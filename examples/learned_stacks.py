"""A LayerStack router learns which stack a position belongs to, and an SFNN trains on its choices.

    python examples/learned_stacks.py [--steps 200]

Synthetic PackedSfenValue records are decoded on the device.  A stack "costs" a
position 1 where it is not the one that the fixed king-rank rule would take, so
the router can be compared with that rule; a trainer would put each stack's loss
there.  The router then evaluates in 8-bit integers and its choices replace the
rule's buckets in an SFNN training step.
"""
import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import bulletou_b200 as bo  # noqa: E402
from bulletou_b200 import synthetic  # noqa: E402
from bulletou_b200.sfnn import HALFKA_HM2_DIMENSIONS, PIECE_INPUTS  # noqa: E402


def main(steps: int = 200, batch: int = 4096, width: int = 16, stacks: int = 9) -> dict:
    if steps < 1:
        raise SystemExit("at least one step is needed")
    ctx = bo.Context(0)
    config = bo.TeacherBatchConfig(feature_set="halfka_hm2", lambda_=1.0, win_rate_model=True)
    producer = bo.TeacherBatchProducer(ctx, config, batch, pinned=False)
    data = producer.new_batch()
    router = bo.StackRouter(ctx, HALFKA_HM2_DIMENSIONS, data.max_active, width, stacks, batch, balance=0.01, seed=1)
    costs = bo.F32Buffer(ctx, batch * stacks)
    learned = bo.I32Buffer(ctx, batch)

    def agreement():
        router.choose(data.stm_indices, learned)
        return float((learned.download() == data.buckets.download()).mean())

    for step in range(steps):
        producer.prepare(ctx, synthetic.psv_records(step, batch), data)
        rule = data.buckets.download()
        costs.upload(1.0 - np.eye(stacks, dtype=np.float32)[rule])
        if step == 0:
            first = agreement()
        router.train_step(bo.RangerUpdateParams(radam=bo.RAdamUpdateParams(step=step + 1, learning_rate=0.01)),
                          data.stm_indices, costs)
        if step % 50 == 0 or step + 1 == steps:
            cost, balance = router.read_losses()
            print(f"step {step}: expected cost {cost:.4f}, balance loss {balance:.5f}, choices {router.read_counts()}")
    producer.prepare(ctx, synthetic.psv_records(10**6, batch), data)  # positions it has not seen
    last = agreement()
    print(f"choices that agree with the rule: {first:.3f} before, {last:.3f} after; by stack {router.read_counts()}")

    shape = bo.SfnnForwardShape(HALFKA_HM2_DIMENSIONS + PIECE_INPUTS, 256, 15, True, 32, stacks)
    weights = synthetic.sfnn_weights(synthetic.rng_for(3), shape.input_size, 256, std=0.05)
    runner = bo.SfnnTrainStepRunner(ctx, bo.SfnnForwardHostWeights(shape, **weights), batch, data.max_active)
    runner.stm_indices, runner.nstm_indices, runner.buckets = data.stm_indices, data.nstm_indices, learned
    runner.targets, runner.entry_weights = data.targets, data.entry_weights
    runner.step_device(ctx, bo.RangerUpdateParams(radam=bo.RAdamUpdateParams(step=1)), bo.ScalarLossKind.SigmoidPow(2.0), 1 / 600)
    loss = runner.read_loss(ctx).mean
    print(f"SFNN step on the learned stacks: loss {loss:.6f}")
    producer.check(ctx)
    return {"before": first, "after": last, "loss": loss, "choices": learned.download()}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    main(parser.parse_args().steps)
