"""MI355X stand-in for the forward and backward pass of reference utils/losses.py (SSDLoss).

Same constructor arguments and the same per-image loss vector as SSDLoss.call
(utils/losses.py:83-181); the gradient with respect to y_pred, which the reference leaves to
TensorFlow's autodiff, is returned explicitly by call_with_grad."""
from ..batched import distill_topk_batch, linear_cross_entropy_batch, ssd_loss_batch


class SSDLoss:
    def __init__(self, neg_pos_ratio=3, n_neg_min=0, alpha=1.0):
        self.neg_pos_ratio = int(neg_pos_ratio)
        self.n_neg_min = int(n_neg_min)
        self.alpha = float(alpha)

    def call(self, y_true, y_pred):
        """(B,) loss per image, utils/losses.py:97-181."""
        return ssd_loss_batch(y_true, y_pred, self.neg_pos_ratio, self.n_neg_min, self.alpha)

    __call__ = call

    def call_with_grad(self, y_true, y_pred):
        """(loss (B,), d mean(loss) / d y_pred (B,A,6))."""
        return ssd_loss_batch(y_true, y_pred, self.neg_pos_ratio, self.n_neg_min, self.alpha,
                              return_grad=True)

    def get_config(self):
        return {"neg_pos_ratio": self.neg_pos_ratio, "n_neg_min": self.n_neg_min, "alpha": self.alpha}


class LinearCrossEntropy:
    """Softmax cross entropy of a linear head over many classes, logits = logit_scale * hidden weight^T, of which
    about 2 GiB are stored at most (an identity head's 10^5 classes, a vocabulary).  No counterpart in the reference, whose heads have two
    classes; arguments and results as batched.linear_cross_entropy_batch."""

    def __init__(self, logit_scale=1.0, label_smoothing=0.0):
        self.logit_scale = float(logit_scale)
        self.label_smoothing = float(label_smoothing)

    def call(self, hidden, weight, labels):
        """(...) loss per row, 0 where the label is negative."""
        return linear_cross_entropy_batch(hidden, weight, labels, self.logit_scale, self.label_smoothing)

    __call__ = call

    def call_with_grad(self, hidden, weight, labels, grad_loss=None):
        """(loss (...), gradients with respect to hidden and weight of mean(loss), or of sum(grad_loss * loss))."""
        return linear_cross_entropy_batch(hidden, weight, labels, self.logit_scale, self.label_smoothing,
                                          grad_loss=grad_loss, return_grad=True)

    def get_config(self):
        return {"logit_scale": self.logit_scale, "label_smoothing": self.label_smoothing}


class TopKDistillation:
    """temperature^2 KL between a teacher's top logits and a student's softmax, such as a small detector's class columns
    taught by a large one's.  No counterpart in the reference; arguments and results as batched.distill_topk_batch."""

    def __init__(self, temperature=1.0):
        self.temperature = float(temperature)

    def call(self, logits, teacher_values, teacher_index, teacher_lse=None):
        """(...) loss per row, 0 where the teacher gives no entry."""
        return distill_topk_batch(logits, teacher_values, teacher_index, self.temperature, teacher_lse)

    __call__ = call

    def call_with_grad(self, logits, teacher_values, teacher_index, teacher_lse=None, grad_loss=None):
        """(loss (...), gradient (..., V) of mean(loss), or of sum(grad_loss * loss))."""
        return distill_topk_batch(logits, teacher_values, teacher_index, self.temperature, teacher_lse,
                                  grad_loss=grad_loss, return_grad=True)

    def get_config(self):
        return {"temperature": self.temperature}
