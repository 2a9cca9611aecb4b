"""Distillation of a student from the largest logits of a teacher."""

import torch.nn as nn

from ..ops import functional as O


class TopKDistillLoss(nn.Module):
    """(1 - alpha) * hard_loss(output, target)
    + alpha * temperature^2 * mean of distill_topk(output, the teacher's top k).

    The teacher's answer is cut to its k largest logits and the sum of the
    rest, as it would be stored; k is lowered to the number of classes.
    temperature^2 keeps the size of the second part's gradient at every
    temperature.
    """

    def __init__(self, hard_loss, k=20, temperature=2.0, alpha=0.5):
        super().__init__()
        assert 0.0 <= alpha <= 1.0
        assert k >= 1 and temperature > 0
        self.hard_loss = hard_loss
        self.k = k
        self.temperature = float(temperature)
        self.alpha = alpha

    def forward(self, output, target, teacher_output):
        answer = O.topk_logits(teacher_output, min(self.k, teacher_output.shape[-1]),
                               self.temperature)
        soft = O.distill_topk(output, *answer, temperature=self.temperature).mean()
        return ((1.0 - self.alpha) * self.hard_loss(output, target)
                + self.alpha * self.temperature ** 2 * soft)
